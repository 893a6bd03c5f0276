// Products of a few rows with 4-bit weights:  y = x W^T (+ bias),  or silu(x Wg^T) * (x Wu^T).
//
//   int4:   W[n, k] = s[n, k / g] (q[n, k] - z[n, k / g]),  q 0..15, z 0..15 (8 if there are none), s bf16, g 32, 64 or 128
//   mxfp4:  W[n, k] = E2M1(c[n, k]) 2^(e[n, k / 32] - 127)
//
// Up to 64 rows the weights' bytes bound it: half a byte a weight, read once.  W is laid out once in the order in which
// the matrix cores take it (v_mfma_f32_16x16x32_bf16, W the A operand, x the B operand): a tile of 16 rows of W and
// 128 values of k is 1 KiB, lane l's 16 bytes the rows' n = l % 16 and, in its dword j, k = 32 j + 8 (l / 16) + 0..7.
// Codes become bf16 in registers, exactly: E2M1 by the scaled conversion with the block's exponent, q by the E4M3
// conversion (the E4M3 numbers of the codes 0 to 15 are code * 2^-9).  A group of int4 is one to four steps of the
// matrix product with its own accumulator a, which then adds s (a - z sum(x)) in fp32; the sums of x come from the same
// instruction with ones for W.
#include "qim_device.h"
#include "qim_runtime.h"

namespace qim {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int FB_WAVES = 8;

struct FourBitWeight {
    const uint8_t *codes, *scales, *zeros;
};
struct FourBitArgs {
    const uint16_t *x;
    int64_t ldx;
    FourBitWeight w[2];  // the second: the up projection of a SwiGLU
    const uint16_t *bias;
    void *out;
    int64_t ldo;
    int M, N, K, KT;     // KT: steps of 128 k
    int f32, wide;       // fp32 output; four values of an output row may be stored at once
};

// The bf16 operand of 8 codes.  E2M1: the block's exponent as the conversion's scale.
__device__ __forceinline__ bf16x8_t fb_e2m1(uint32_t w, float scale) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// int4: the low halves of the four bytes, then the high ones.
__device__ __forceinline__ bf16x8_t fb_int4(uint32_t w) {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    const float s = 512.0f;
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The operand of q - z itself, for rows that hold values whose product with q alone leaves fp32 (infinities among
// them): q x - z x would be NaN or infinite where (q - z) x is not.
__device__ __forceinline__ bf16x8_t fb_int4_centred(uint32_t w, int z) {
    bf16x8_t v;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int q = (int)((w >> (i < 4 ? 8 * i : 8 * (i - 4) + 4)) & 15u);
        v[i] = (__bf16)(float)(q - z);
    }
    return v;
}
__device__ __forceinline__ bf16x8_t fb_ones() {
    const u32x4_t w = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    return __builtin_bit_cast(bf16x8_t, w);
}

// One workgroup: NT tiles of 16 output columns (with SWIGLU: the same tile of both weights, NT = 2) and 16 NR rows;
// its waves take the steps of 128 k in turn and join in LDS.  G: groups of int4 in a step, 0 for mxfp4.
template <int G, int NT, int NR, bool SWIGLU>
__global__ __launch_bounds__(64 * FB_WAVES) void k_fourbit(FourBitArgs p) {
    __shared__ f32x4_t part[FB_WAVES][NT * NR][64];
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row0 = blockIdx.y * 16 * NR;
    int64_t tile[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) tile[i] = SWIGLU ? blockIdx.x : (int64_t)blockIdx.x * NT + i;
    const int ntiles = (p.N + 15) / 16;
#pragma unroll
    for (int i = 0; i < NT; ++i) tile[i] = tile[i] < ntiles ? tile[i] : ntiles - 1;  // (repeated, not stored)

    f32x4_t acc[NT][NR];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[i][r] = f32x4_t{};
    auto steps = [&](auto centred, f32x4_t (&acc)[NT][NR]) {
        constexpr bool CENTRED = decltype(centred)::value;
        for (int t = wave; t < p.KT; t += FB_WAVES) {
            uint4 x[NR][4];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int row = row0 + 16 * r + lr;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k = 128 * t + 32 * j + 8 * kg;
                    x[r][j] = row < p.M && k < p.K ? *reinterpret_cast<const uint4 *>(p.x + row * p.ldx + k) : make_uint4(0, 0, 0, 0);
                }
            }
            f32x4_t xs[NR][G ? G : 1];
            if constexpr (G > 0 && !CENTRED) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        xs[r][j * G / 4] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            fb_ones(), __builtin_bit_cast(bf16x8_t, x[r][j]), j % (4 / G) ? xs[r][j * G / 4] : f32x4_t{}, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const FourBitWeight &w = p.w[SWIGLU ? i : 0];
                const int64_t at = tile[i] * p.KT + t;
                const uint4 c4 = *reinterpret_cast<const uint4 *>(w.codes + at * 1024 + lane * 16);
                const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
                if constexpr (G == 0) {
                    const uint32_t e = *reinterpret_cast<const uint32_t *>(w.scales + (at * 16 + lr) * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bf16x8_t a = fb_e2m1(c[j], mx_scale_operand((int)((e >> (8 * j)) & 0xffu)));
#pragma unroll
                        for (int r = 0; r < NR; ++r)
                            acc[i][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8_t, x[r][j]), acc[i][r], 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const uint2 s2 = *reinterpret_cast<const uint2 *>(w.scales + ((at * G + g) * 16 + 4 * kg) * 2);
                        const float s[4] = {bf_lo(s2.x), bf_hi(s2.x), bf_lo(s2.y), bf_hi(s2.y)};
                        const uint32_t z4 = w.zeros ? *reinterpret_cast<const uint32_t *>(w.zeros + (at * G + g) * 16 + 4 * kg) : 0x08080808u;
                        const int zn = CENTRED ? (w.zeros ? w.zeros[(at * G + g) * 16 + lr] : 8) : 0;
                        f32x4_t a[NR];
#pragma unroll
                        for (int j = g * (4 / G); j < (g + 1) * (4 / G); ++j) {
                            const bf16x8_t v = CENTRED ? fb_int4_centred(c[j], zn) : fb_int4(c[j]);
#pragma unroll
                            for (int r = 0; r < NR; ++r)
                                a[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8_t, x[r][j]),
                                                                                j % (4 / G) ? a[r] : f32x4_t{}, 0, 0, 0);
                        }
#pragma unroll
                        for (int r = 0; r < NR; ++r)
#pragma unroll
                            for (int n = 0; n < 4; ++n) {
                                const float y = CENTRED ? a[r][n] : __builtin_fmaf(-(float)((z4 >> (8 * n)) & 0xffu), xs[r][g][n], a[r][n]);
                                acc[i][r][n] = __builtin_fmaf(s[n], y, acc[i][r][n]);
                            }
                    }
                }
            }
        }
    };
    steps(std::false_type{}, acc);
    if constexpr (G > 0) {
        bool finite = true;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
                for (int n = 0; n < 4; ++n) finite = finite && acc[i][r][n] - acc[i][r][n] == 0.0f;
        if (__builtin_amdgcn_ballot_w64(!finite)) {  // the values that are finite keep their bits
            f32x4_t again[NT][NR];
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < NR; ++r) again[i][r] = f32x4_t{};
            steps(std::true_type{}, again);
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        acc[i][r][n] = acc[i][r][n] - acc[i][r][n] == 0.0f ? acc[i][r][n] : again[i][r][n];
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < NR; ++r) part[wave][i * NR + r][lane] = acc[i][r];
    __syncthreads();
    constexpr int OUT = SWIGLU ? NR : NT * NR;  // 16 x 16 blocks of output
    for (int i = tid; i < OUT * 64; i += 64 * FB_WAVES) {
        const int blk = i >> 6, l = i & 63;
        f32x4_t y = {}, u = {};
#pragma unroll
        for (int v = 0; v < FB_WAVES; ++v) {
            y += part[v][blk][l];
            if (SWIGLU) u += part[v][NR + blk][l];
        }
        const int64_t ct = SWIGLU ? blockIdx.x : (int64_t)blockIdx.x * NT + blk / NR;
        const int64_t n0 = ct * 16 + 4 * (l >> 4);
        const int row = row0 + 16 * (blk % NR) + (l & 15);
        if (row >= p.M || n0 >= p.N) continue;
        const int left = p.N - n0 < 4 ? (int)(p.N - n0) : 4;
        if (SWIGLU) {
#pragma unroll
            for (int n = 0; n < 4; ++n) y[n] = y[n] / (1.0f + __builtin_amdgcn_exp2f(-1.44269504f * y[n])) * u[n];
        } else if (p.bias) {
            for (int n = 0; n < left; ++n) y[n] += bf16_to_f32(p.bias[n0 + n]);
        }
        if (p.f32) {
            float *o = static_cast<float *>(p.out) + row * p.ldo + n0;
            if (p.wide && left == 4) *reinterpret_cast<f32x4_t *>(o) = y;
            else
                for (int n = 0; n < left; ++n) o[n] = y[n];
        } else {
            uint16_t *o = static_cast<uint16_t *>(p.out) + row * p.ldo + n0;
            const uint32_t a = pack_bf16x2(y[0], y[1]), b = pack_bf16x2(y[2], y[3]);
            if (p.wide && left == 4) *reinterpret_cast<uint2 *>(o) = make_uint2(a, b);
            else
                for (int n = 0; n < left; ++n) o[n] = (uint16_t)((n < 2 ? a : b) >> (16 * (n & 1)));
        }
    }
}

template <int G, bool SWIGLU>
static void launch_fourbit(const FourBitArgs &a, hipStream_t st) {
    const int nt = (a.N + 15) / 16, rows = a.M > 32 ? 4 : a.M > 16 ? 2 : 1;
    const dim3 grid((unsigned)nt, (unsigned)((a.M + 16 * rows - 1) / (16 * rows)));
    constexpr int NT = SWIGLU ? 2 : 1;
    launch(rows == 4 ? k_fourbit<G, NT, 4, SWIGLU> : rows == 2 ? k_fourbit<G, NT, 2, SWIGLU> : k_fourbit<G, NT, 1, SWIGLU>, grid,
           dim3(64 * FB_WAVES), 0, st, a);
}

}  // namespace qim

using namespace qim;

extern "C" int qim_fourbit_matmul(const void *x, int64_t ldx, int group, const void *codes, const void *scales, const void *zeros,
                                  const void *codes2, const void *scales2, const void *zeros2, const void *bias, void *out,
                                  int64_t ldo, int out_f32, int64_t M, int64_t N, int64_t K, void *stream) {
    const char *who = "qim_fourbit_matmul";
    QIM_REQUIRE(x && codes && scales && out && !codes2 == !scales2, QIM_ERR_ARG, "%s: null pointer", who);
    QIM_REQUIRE(group == 0 || group == 32 || group == 64 || group == 128, QIM_ERR_ARG, "%s: group %d (0 for mxfp4, 32, 64, 128)", who, group);
    QIM_REQUIRE((group || (!zeros && !zeros2)) && (codes2 ? !zeros == !zeros2 : !zeros2), QIM_ERR_ARG,
                "%s: zero points go with int4, and with both weights or none", who);
    QIM_REQUIRE(!codes2 || !bias, QIM_ERR_ARG, "%s: no bias with the SwiGLU", who);
    QIM_REQUIRE(out_f32 == 0 || out_f32 == 1, QIM_ERR_ARG, "%s: out_f32 %d", who, out_f32);
    QIM_REQUIRE(M > 0 && N > 0 && K > 0 && K % (group ? group : 32) == 0 && M < (1 << 20) && N < (1 << 24) && K < (1 << 24),
                QIM_ERR_SHAPE, "%s: M %lld, N %lld, K %lld in groups of %d", who, (long long)M, (long long)N, (long long)K, group ? group : 32);
    QIM_REQUIRE(ldx >= K && ldx % 8 == 0 && ldo >= N && aligned16(x) && aligned16(codes) && aligned16(scales) && aligned16(zeros) &&
                    aligned16(codes2) && aligned16(scales2) && aligned16(zeros2) &&
                    (reinterpret_cast<uintptr_t>(out) & (out_f32 ? 3u : 1u)) == 0 && (reinterpret_cast<uintptr_t>(bias) & 1u) == 0,
                QIM_ERR_LAYOUT, "%s: rows of x must be 16-byte aligned", who);
    const int64_t size = out_f32 ? 4 : 2;
    QIM_REQUIRE(!bytes_share(out, size * ((M - 1) * ldo + N), x, 2 * ((M - 1) * ldx + K)), QIM_ERR_ARG, "%s: out overlaps x", who);
    FourBitArgs a{(const uint16_t *)x, ldx,
                  {{(const uint8_t *)codes, (const uint8_t *)scales, (const uint8_t *)zeros},
                   {(const uint8_t *)codes2, (const uint8_t *)scales2, (const uint8_t *)zeros2}},
                  (const uint16_t *)bias, out, ldo, (int)M, (int)N, (int)K, (int)((K + 127) / 128), out_f32,
                  ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * size - 1)) == 0};
    hipStream_t st = as_stream(stream);
    switch ((codes2 ? 4 : 0) + (group ? 128 / group == 4 ? 3 : 128 / group : 0)) {
        case 0: launch_fourbit<0, false>(a, st); break;
        case 1: launch_fourbit<1, false>(a, st); break;
        case 2: launch_fourbit<2, false>(a, st); break;
        case 3: launch_fourbit<4, false>(a, st); break;
        case 4: launch_fourbit<0, true>(a, st); break;
        case 5: launch_fourbit<1, true>(a, st); break;
        case 6: launch_fourbit<2, true>(a, st); break;
        default: launch_fourbit<4, true>(a, st); break;
    }
    return check_launch(who);
}
