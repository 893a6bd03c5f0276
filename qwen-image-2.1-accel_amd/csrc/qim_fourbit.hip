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
// matrix product with its own accumulator, which one more product then corrects for the zero points: z times the negated
// sum of x as three bf16 terms (24 bits), the sums of x coming from the same instruction with ones for W.  The group's
// scale enters in fp32.
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

// The zero points' product: B is minus the sum of x (of this lane's row, in all four values of xs) as three bf16 terms in
// the first values of k, A is z (of this lane's row of W) in the same places.  The instruction is the one that summed the
// group: behind it a shorter shape on the same accumulator needs wait states that hipcc of ROCm 7.2 does not
// put in (16x16x16 three instructions later read two of the four sums too early).
__device__ __forceinline__ bf16x8_t fb_negated_sum(const f32x4_t &xs, int kg) {
    const float v = -xs[0], hi = rbf(v), mid = rbf(v - hi);
    const uint32_t lo = kg == 0 ? pack_bf16x2(hi, mid) : 0u, up = kg == 0 ? pack_bf16x2((v - hi) - mid, 0.0f) : 0u;
    return __builtin_bit_cast(bf16x8_t, u32x4_t{lo, up, 0, 0});
}
__device__ __forceinline__ bf16x8_t fb_zero_point(uint32_t z) {
    const uint32_t b = __float_as_uint((float)z) >> 16;
    return __builtin_bit_cast(bf16x8_t, u32x4_t{b | (b << 16), b, 0, 0});
}

// Four values of an output row from column n0 on (those that exist), through the epilogue.
template <bool SWIGLU>
__device__ __forceinline__ void fb_store(const FourBitArgs &p, int64_t row, int64_t n0, f32x4_t y, f32x4_t u) {
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
    // What a step reads; the next one's is on its way while one is multiplied.
    struct Step {
        uint4 x[NR][4], w[NT], s[NT][G == 4 ? 2 : 1];  // s: the scales of rows 4 kg .. 4 kg + 3, by group (G 1: half of it)
        uint32_t z[NT];                                // mxfp4: the exponents, by j; int4: the zero points, by group
    };
    auto load = [&](Step &v, int t) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const FourBitWeight &w = p.w[SWIGLU ? i : 0];
            const int64_t at = tile[i] * p.KT + t;
            v.w[i] = *reinterpret_cast<const uint4 *>(w.codes + at * 1024 + lane * 16);
            if constexpr (G == 0) {
                v.z[i] = *reinterpret_cast<const uint32_t *>(w.scales + (at * 16 + lr) * 4);
            } else {
                const uint8_t *sc = w.scales + (at * 4 + kg) * (8 * G), *z = w.zeros + (at * 16 + lr) * G;
                if constexpr (G == 1) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(sc);
                    v.s[i][0] = make_uint4(u.x, u.y, 0, 0);
                } else {
#pragma unroll
                    for (int g = 0; g < G / 2; ++g) v.s[i][g] = reinterpret_cast<const uint4 *>(sc)[g];
                }
                v.z[i] = 0x08080808u;
                if (w.zeros) v.z[i] = G == 4 ? *reinterpret_cast<const uint32_t *>(z) : G == 2 ? *reinterpret_cast<const uint16_t *>(z) : *z;
            }
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = row0 + 16 * r + lr;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = 128 * t + 32 * j + 8 * kg;
                v.x[r][j] = row < p.M && k < p.K ? *reinterpret_cast<const uint4 *>(p.x + row * p.ldx + k) : make_uint4(0, 0, 0, 0);
            }
        }
    };
    auto multiply = [&](const Step &v, auto centred, f32x4_t (&acc)[NT][NR]) {
        constexpr bool CENTRED = decltype(centred)::value;
        auto word = [](const uint4 &u, int j) { return j == 0 ? u.x : j == 1 ? u.y : j == 2 ? u.z : u.w; };
        if constexpr (G == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const bf16x8_t a = fb_e2m1(word(v.w[i], j), mx_scale_operand((int)((v.z[i] >> (8 * j)) & 0xffu)));
#pragma unroll
                    for (int r = 0; r < NR; ++r)
                        acc[i][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8_t, v.x[r][j]), acc[i][r], 0, 0, 0);
                }
        } else {
            constexpr int PER = 4 / G;  // matrix steps of a group
#pragma unroll
            for (int g = 0; g < G; ++g) {
                bf16x8_t xb[NR];
                if constexpr (!CENTRED) {
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        f32x4_t xs = {};
#pragma unroll
                        for (int j = g * PER; j < (g + 1) * PER; ++j)
                            xs = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb_ones(), __builtin_bit_cast(bf16x8_t, v.x[r][j]), xs, 0, 0, 0);
                        xb[r] = fb_negated_sum(xs, kg);
                    }
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const uint32_t s0 = word(v.s[i][g / 2], 2 * (g & 1)), s1 = word(v.s[i][g / 2], 2 * (g & 1) + 1), z = (v.z[i] >> (8 * g)) & 0xffu;
                    const float s[4] = {bf_lo(s0), bf_hi(s0), bf_lo(s1), bf_hi(s1)};
                    f32x4_t a[NR];
#pragma unroll
                    for (int j = g * PER; j < (g + 1) * PER; ++j) {
                        const bf16x8_t w = CENTRED ? fb_int4_centred(word(v.w[i], j), (int)z) : fb_int4(word(v.w[i], j));
#pragma unroll
                        for (int r = 0; r < NR; ++r)
                            a[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, __builtin_bit_cast(bf16x8_t, v.x[r][j]), j % PER ? a[r] : f32x4_t{}, 0, 0, 0);
                    }
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        if constexpr (!CENTRED) a[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb_zero_point(z), xb[r], a[r], 0, 0, 0);
#pragma unroll
                        for (int n = 0; n < 4; ++n) acc[i][r][n] = __builtin_fmaf(s[n], a[r][n], acc[i][r][n]);
                    }
                }
            }
        }
    };
    auto steps = [&](auto centred, f32x4_t (&acc)[NT][NR]) {
        int t = wave;
        if (t >= p.KT) return;
        Step a, b;
        load(a, t);
        for (;;) {
            if (t + FB_WAVES < p.KT) load(b, t + FB_WAVES);
            multiply(a, centred, acc);
            if ((t += FB_WAVES) >= p.KT) break;
            if (t + FB_WAVES < p.KT) load(a, t + FB_WAVES);
            multiply(b, centred, acc);
            if ((t += FB_WAVES) >= p.KT) break;
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
        fb_store<SWIGLU>(p, row, n0, y, u);
    }
}

// Many rows: a workgroup of 2 x 2 waves, each with WM tiles of 16 rows of x and WN of 16 columns; x goes through LDS in
// steps of 128 k (two buffers, 16-byte chunk c of row r at c ^ (r % 16), so that the 16 rows of an operand read lie in
// different banks), the weights straight from memory to the registers of the waves that multiply with them.
// int4's scales and zero points go through LDS beside x.
template <int G, int WM, int WN, bool SWIGLU>
__global__ __launch_bounds__(256, 2) void k_fourbit_tile(FourBitArgs p, uint32_t ncol) {
    constexpr int ROWS = 32 * WM, CH = ROWS * 16 / 256;   // 16-byte chunks of a step per lane
    extern __shared__ __attribute__((aligned(1024))) uint4 fb_lds[];
    uint4 (*const xt)[ROWS * 16] = reinterpret_cast<uint4 (*)[ROWS * 16]>(fb_lds);
    constexpr int SB = 2 * G * 16, ZB = G * 16, TILES = 2 * WN;   // bytes of scales and of zero points of a tile's step
    uint8_t (*const st)[TILES * (SB + ZB)] = reinterpret_cast<uint8_t (*)[TILES * (SB + ZB)]>(fb_lds + 2 * ROWS * 16);
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave & 1, wn = wave >> 1;
    const uint32_t col = blockIdx.x % ncol;
    const int64_t row0 = (int64_t)(blockIdx.x / ncol) * ROWS;
    const int64_t ntiles = (p.N + 15) / 16;
    constexpr int OT = SWIGLU ? WN / 2 : WN;              // column tiles of output a wave
    const int64_t tile0 = ((int64_t)col * 2 + wn) * OT;

    f32x4_t acc[WN][WM];
    auto run = [&](auto centred) {
        constexpr bool CENTRED = decltype(centred)::value;
#pragma unroll
        for (int i = 0; i < WN; ++i)
#pragma unroll
            for (int r = 0; r < WM; ++r) acc[i][r] = f32x4_t{};
        uint4 wc[WN];
        // A step of x to LDS, 1 KiB a wave and instruction: lane l brings chunk (l % 16) ^ (r % 16) of row r = its
        // quarter's.  Chunks past the end (rows, and k of the last step) bring others instead; nothing multiplies with them.
        auto load = [&](int t) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int r = (wave * CH + i) * 4 + kg, k = 128 * t + 8 * (lr ^ (r & 15));
                const int64_t row = row0 + r < p.M ? row0 + r : p.M - 1;
                const uint16_t *src = p.x + row * p.ldx + (k < p.K ? k : 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                                 (__attribute__((address_space(3))) void *)&xt[t & 1][(wave * CH + i) * 64], 16, 0, 0);
            }
        };
        auto at_of = [&](int i, int t) {
            const int64_t tl = tile0 + (SWIGLU ? i >> 1 : i);
            return (tl < ntiles ? tl : ntiles - 1) * p.KT + t;
        };
        auto load_w = [&](int t) {
#pragma unroll
            for (int i = 0; i < WN; ++i)
                wc[i] = *reinterpret_cast<const uint4 *>(p.w[SWIGLU ? i & 1 : 0].codes + at_of(i, t) * 1024 + lane * 16);
        };
        // int4: the scales of all the workgroup's tiles, then the zero points, in 16-byte pieces to the first lanes.
        constexpr int NS = TILES * SB / 16, NZ = TILES * ZB / 16;
        static_assert(NS + NZ <= 256, "a piece a lane");
        uint4 piece = make_uint4(0x08080808u, 0x08080808u, 0x08080808u, 0x08080808u);
        auto load_s = [&](int t) {
            if constexpr (G > 0) {
                constexpr int PS = SB / 16, PZ = ZB / 16;
                if (tid < NS + NZ) {
                    const bool sc = tid < NS;
                    const int q = sc ? tid : tid - NS, i = sc ? q / PS : q / PZ, in = sc ? q % PS : q % PZ;
                    const int64_t tl = (int64_t)col * 2 * OT + (SWIGLU ? (i / WN) * OT + (i % WN) / 2 : i);
                    const FourBitWeight &fw = p.w[SWIGLU ? i & 1 : 0];
                    const int64_t at = (tl < ntiles ? tl : ntiles - 1) * p.KT + t;
                    if (sc) piece = reinterpret_cast<const uint4 *>(fw.scales + at * SB)[in];
                    else if (fw.zeros) piece = reinterpret_cast<const uint4 *>(fw.zeros + at * ZB)[in];
                }
            }
        };
        load(0);
        load_w(0);
        load_s(0);
        for (int t = 0; t < p.KT; ++t) {
            if constexpr (G > 0) {
                if (tid < NS + NZ) reinterpret_cast<uint4 *>(st[t & 1])[tid] = piece;
            }
            const uint4 *const buf = xt[t & 1];
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's part of the step is in LDS
            __syncthreads();                                  // every wave's is, and the other buffer has been read
            uint4 w[WN];
#pragma unroll
            for (int i = 0; i < WN; ++i) w[i] = wc[i];
            if (t + 1 < p.KT) {
                load(t + 1);
                load_w(t + 1);
                load_s(t + 1);
            }
            uint32_t e[WN];
            if constexpr (G == 0) {
#pragma unroll
                for (int i = 0; i < WN; ++i) e[i] = *reinterpret_cast<const uint32_t *>(p.w[SWIGLU ? i & 1 : 0].scales + (at_of(i, t) * 16 + lr) * 4);
            }
            constexpr int PER = G ? 4 / G : 1;            // matrix steps of a group
#pragma unroll
            for (int g = 0; g < 4 / PER; ++g) {
                if (128 * t + 32 * PER * g >= p.K) break;  // the last step
                uint32_t zn[WN];
                float sc[WN][4];
                if constexpr (G > 0) {
#pragma unroll
                    for (int i = 0; i < WN; ++i) {
                        const int tl = wn * WN + i;
                        const uint2 s2 = *reinterpret_cast<const uint2 *>(st[t & 1] + tl * SB + (kg * G + g) * 8);
                        sc[i][0] = bf_lo(s2.x), sc[i][1] = bf_hi(s2.x), sc[i][2] = bf_lo(s2.y), sc[i][3] = bf_hi(s2.y);
                        zn[i] = st[t & 1][TILES * SB + tl * ZB + lr * G + g];
                    }
                }
                f32x4_t a[WN][WM], xs[WM];
#pragma unroll
                for (int j = g * PER; j < (g + 1) * PER; ++j) {
                    bf16x8_t xf[WM];
#pragma unroll
                    for (int r = 0; r < WM; ++r) {
                        const int row = (wm * WM + r) * 16 + lr;
                        xf[r] = __builtin_bit_cast(bf16x8_t, buf[row * 16 + ((4 * j + kg) ^ lr)]);
                    }
                    if constexpr (G > 0 && !CENTRED) {
#pragma unroll
                        for (int r = 0; r < WM; ++r)
                            xs[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb_ones(), xf[r], j % PER ? xs[r] : f32x4_t{}, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < WN; ++i) {
                        const uint32_t c = j == 0 ? w[i].x : j == 1 ? w[i].y : j == 2 ? w[i].z : w[i].w;
                        const bf16x8_t wf = G == 0 ? fb_e2m1(c, mx_scale_operand((int)((e[i] >> (8 * j)) & 0xffu)))
                                                   : CENTRED ? fb_int4_centred(c, (int)zn[i]) : fb_int4(c);
#pragma unroll
                        for (int r = 0; r < WM; ++r) {
                            if constexpr (G == 0) acc[i][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[r], acc[i][r], 0, 0, 0);
                            else a[i][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[r], j % PER ? a[i][r] : f32x4_t{}, 0, 0, 0);
                        }
                    }
                }
                if constexpr (G > 0) {
                    if constexpr (!CENTRED) {
                        bf16x8_t xb[WM];
#pragma unroll
                        for (int r = 0; r < WM; ++r) xb[r] = fb_negated_sum(xs[r], kg);
#pragma unroll
                        for (int i = 0; i < WN; ++i)
#pragma unroll
                            for (int r = 0; r < WM; ++r)
                                a[i][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb_zero_point(zn[i]), xb[r], a[i][r], 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < WN; ++i)
#pragma unroll
                        for (int r = 0; r < WM; ++r)
#pragma unroll
                            for (int n = 0; n < 4; ++n) acc[i][r][n] = __builtin_fmaf(sc[i][n], a[i][r][n], acc[i][r][n]);
                }
            }
        }
        __syncthreads();  // the buffers are free
    };
    // `only`: the values to store, a bit for each four.
    auto store = [&](uint64_t only) {
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
            for (int r = 0; r < WM; ++r) {
                const int64_t row = row0 + (wm * WM + r) * 16 + lr, n0 = (tile0 + i) * 16 + 4 * kg;
                if (row < p.M && n0 < p.N && ((only >> (i * WM + r)) & 1)) {
                    if constexpr (SWIGLU) fb_store<true>(p, row, n0, acc[2 * i][r], acc[2 * i + 1][r]);
                    else fb_store<false>(p, row, n0, acc[i][r], f32x4_t{});
                }
            }
    };
    run(std::false_type{});
    uint64_t bad = 0;
    if constexpr (G > 0) {
#pragma unroll
        for (int i = 0; i < WN; ++i)
#pragma unroll
            for (int r = 0; r < WM; ++r)
#pragma unroll
                for (int n = 0; n < 4; ++n) bad |= (uint64_t)!(acc[i][r][n] - acc[i][r][n] == 0.0f) << ((SWIGLU ? i >> 1 : i) * WM + r);
    }
    store(~bad);
    if constexpr (G > 0) {
        uint32_t *const flag = reinterpret_cast<uint32_t *>(xt);
        const uint64_t any = __builtin_amdgcn_ballot_w64(bad != 0);
        if (lane == 0) flag[wave] = any != 0;
        __syncthreads();
        const uint32_t again = flag[0] | flag[1] | flag[2] | flag[3];
        __syncthreads();
        if (again) {
            run(std::true_type{});
            store(bad);
        }
    }
}

template <int G, bool SWIGLU>
static int launch_fourbit(const FourBitArgs &a, hipStream_t st) {
    const int64_t ntiles = (a.N + 15) / 16;
    if (a.M > 64) {
#ifndef FB_WM
#define FB_WM 4
#define FB_WN 4
#endif
        constexpr int cols = 2 * (SWIGLU ? FB_WN / 2 : FB_WN);
        const uint32_t ncol = (uint32_t)((ntiles + cols - 1) / cols);
        constexpr int bytes = 2 * (32 * FB_WM * 256 + 2 * FB_WN * 3 * G * 16);
        static std::atomic<bool> done[QIM_MAX_DEVICES];
        const int rc = reserve_lds(reinterpret_cast<const void *>(k_fourbit_tile<G, FB_WM, FB_WN, SWIGLU>), bytes, done, "qim_fourbit_matmul");
        if (rc != QIM_OK) return rc;
        launch(k_fourbit_tile<G, FB_WM, FB_WN, SWIGLU>, dim3(ncol * (unsigned)((a.M + 32 * FB_WM - 1) / (32 * FB_WM))), dim3(256), bytes, st, a, ncol);
        return QIM_OK;
    }
    const int nt = (int)ntiles, rows = a.M > 32 ? 4 : a.M > 16 ? 2 : 1;
    const dim3 grid((unsigned)nt, (unsigned)((a.M + 16 * rows - 1) / (16 * rows)));
    constexpr int NT = SWIGLU ? 2 : 1;
    launch(rows == 4 ? k_fourbit<G, NT, 4, SWIGLU> : rows == 2 ? k_fourbit<G, NT, 2, SWIGLU> : k_fourbit<G, NT, 1, SWIGLU>, grid,
           dim3(64 * FB_WAVES), 0, st, a);
    return QIM_OK;
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
    int rc;
    switch ((codes2 ? 4 : 0) + (group ? 128 / group == 4 ? 3 : 128 / group : 0)) {
        case 0: rc = launch_fourbit<0, false>(a, st); break;
        case 1: rc = launch_fourbit<1, false>(a, st); break;
        case 2: rc = launch_fourbit<2, false>(a, st); break;
        case 3: rc = launch_fourbit<4, false>(a, st); break;
        case 4: rc = launch_fourbit<0, true>(a, st); break;
        case 5: rc = launch_fourbit<1, true>(a, st); break;
        case 6: rc = launch_fourbit<2, true>(a, st); break;
        default: rc = launch_fourbit<4, true>(a, st); break;
    }
    return rc != QIM_OK ? rc : check_launch(who);
}
