// Products of a few rows with 4-bit weights:  y = x W^T (+ bias),  or silu(x Wg^T) * (x Wu^T).
//
//   int4:   W[n, k] = s[n, k / g] (q[n, k] - z[n, k / g]),  q 0..15, z 0..15 (8 if there are none), s bf16, g 32, 64 or 128
//   mxfp4:  W[n, k] = E2M1(c[n, k]) 2^(e[n, k / 32] - 127)
//
// Up to some 16 rows the weights' bytes bound it: half a byte a weight, read once; beyond, the vector instructions that make
// operands of codes and, for int4, take the groups' scales in.  W is laid out once in the order in which the matrix cores take it
// (v_mfma_f32_16x16x32_bf16, W the A operand, x the B operand): a tile of 16 rows of W and a step of 128 k is 1 KiB, lane
// l's 16 bytes the row n = l % 16 and, in its dword j, k = 32 j + 8 (l / 16) + 0..7.  Codes become bf16 in registers, exactly:
// E2M1 by the scaled conversion with the block's exponent; q - z by a table of the 16 E4M3 codes of 0 - z .. 15 - z (|q - z| is
// at most 15, which 4 significand bits hold), looked up four codes at a time by v_perm, and the E4M3 conversion.  A
// group of int4 is one to four steps of the product with an accumulator of its own, which enters the row's in fp32, times the
// group's scale.  q - z enters times 2^-11, which the last sum takes back (exact): a group's sum before its scale, up to
// 15 * 128 times the row's largest value, then is in fp32 whatever x holds (and results below 2^-114 are off by some 2^-138).
// (Taking q for q - z and z times the sum of x away again in fp32 costs less per code and
// more per group and row; it also makes NaN of infinities.)
//
// Two kernels.  k_fourbit, few rows or few columns: the waves of a workgroup take the steps of k in turn, each for the whole
// tile of output and through a ring in LDS of its own, and join at the end; no barrier stands in the loop.  k_fourbit_tile,
// the others: stages in LDS that eight waves share, and up to 128 rows for every operand made of codes.
// Measured (calls one behind the other; from a graph 1-3 us more): int4 g 128, 1 row, 4096 -> 12288 9.0 us, 2.9 TB/s; mxfp4, 16 rows,
// 12288 -> 4096 9.1 us, 3.0 TB/s; int4 g 64, 24 rows, 4096 -> 12288 SwiGLU 20.8 us; int4 g 32, 154 rows, 4096 -> 12288 36 us, 430
// TFLOP/s; mxfp4, 1024 rows, 4096 -> 4096 38.5 us, 890 TFLOP/s.
#include "qim_device.h"
#include "qim_runtime.h"

namespace qim {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr float FB_UNIT = 0x1p-11f;  // of int4's operands

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
// int4: byte i of w holds code i in its low and code i + 4 in its high half; t the E4M3 codes (times 2^-9) of q - z for
// q 0..15.  A byte permutation chooses among 8: both halves of the table, then between them by the code's high bit.
__device__ __forceinline__ bf16x8_t fb_int4(uint32_t w, const uint4 &t) {
    auto look = [&](uint32_t v) {
        const uint32_t low = v & 0x07070707u, half = ((v >> 1) & 0x04040404u) | 0x03020100u;
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(t.w, t.z, low), __builtin_amdgcn_perm(t.y, t.x, low), half);
    };
    const uint32_t lo = look(w), hi = look(w >> 4);
    const float s = 512.0f * FB_UNIT;
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The table of z: byte q is |q - z|, with the sign bit where q < z.
__device__ __forceinline__ uint32_t fb_table(int z, int first) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = first + i - z;
        w |= (uint32_t)(d < 0 ? 0x80 | -d : d) << (8 * i);
    }
    return w;
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

__device__ __forceinline__ uint32_t fb_word(const uint4 &u, int j) { return j == 0 ? u.x : j == 1 ? u.y : j == 2 ? u.z : u.w; }

// LDS DMA that the compiler does not see as a write of LDS (it would wait for all of them before every read): lane i's 16
// bytes land at lds + 16 i.  The stages' own waits and barriers order them; the s_nop covers the wait state between the
// write of M0 and its use.
__device__ __forceinline__ void fb_dma(const uint8_t *base, uint32_t off, uint32_t lds) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}
template <int N>
__device__ __forceinline__ void fb_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// 4 RX rows and NT tiles of 16 columns of W (SWIGLU: NT / 2 of each weight) a workgroup, whose waves take the steps of k
// in turn.  G: groups of int4 in a step, 0 for mxfp4.  Everything goes through a ring of S stages in LDS of the wave's own:
// S steps are on their way without registers held for them, and x, whose rows an operand takes from 16 places at
// once, arrives in whole 256-byte rows (read by the operands' lanes themselves, 16 bytes here and there, it cost four
// times as many requests as bytes and more time than W).  No barrier stands in the loop.
template <int G, int NT, int RX, int WAVES, int S>
struct FbRing {
    static constexpr int SB = G ? 32 * G : 64, ZB = 16 * G;  // bytes of a tile's scales or exponents, and of its zero points
    static constexpr int CODES = RX * 1024, SCALES = CODES + NT * 1024, ZEROS = SCALES + NT * SB, BYTES = (ZEROS + NT * ZB + 15) / 16 * 16;
    static constexpr int LOADS = RX + NT * (G ? 3 : 2);
    static constexpr int JOIN = WAVES * NT * 1024, TABLES = WAVES * S * BYTES > JOIN ? WAVES * S * BYTES : JOIN, LDS = TABLES + (G ? 256 : 0);
};
template <int G, int NT, int RX, int WAVES, int S, bool SWIGLU>
__global__ __launch_bounds__(64 * WAVES, 4) void k_fourbit(FourBitArgs p) {
    using Ring = FbRing<G, NT, RX, WAVES, S>;
    constexpr int OT = SWIGLU ? NT / 2 : NT;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    uint4 *const tables = reinterpret_cast<uint4 *>(lds + Ring::TABLES);
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ntiles = (p.N + 15) / 16;
    const int row0 = (int)blockIdx.y * 4 * RX, rows = p.M - row0;
    const uint8_t *const x0 = reinterpret_cast<const uint8_t *>(p.x + row0 * p.ldx);
    const uint8_t *const ring = lds + wave * (S * Ring::BYTES);
    const uint32_t ring0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)ring;
    // Rows and tiles past the last are the last (computed, not stored); a 16-byte chunk c of row r of x lies at c ^ r, so that
    // the rows of an operand lie in different banks.
    uint32_t xoff[RX];
#pragma unroll
    for (int i = 0; i < RX; ++i) {
        const int r = 4 * i + kg;
        xoff[i] = (uint32_t)(r < rows ? r : rows - 1) * (uint32_t)(2 * p.ldx) + 16 * (lr ^ r);
    }
    auto issue = [&](int t, int slot) {
        const uint32_t to = ring0 + slot * Ring::BYTES;
        const uint8_t *const xt = x0 + (int64_t)t * 256;
        const bool whole = 128 * t + 128 <= p.K;
#pragma unroll
        for (int i = 0; i < RX; ++i) {
            uint32_t off = xoff[i];
            if (!whole) {  // k past the end: others come, and nothing multiplies with them
                const int k = 8 * (lr ^ (4 * i + kg));
                off -= 128 * t + k < p.K ? 0 : 2 * k;
            }
            fb_dma(xt, off, to + i * 1024);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const FourBitWeight &w = p.w[SWIGLU ? i & 1 : 0];
            const int tl = (int)blockIdx.x * OT + (SWIGLU ? i >> 1 : i);
            const int64_t at = (int64_t)(tl < ntiles ? tl : ntiles - 1) * p.KT + t;
            fb_dma(w.codes + at * 1024, lane * 16, to + Ring::CODES + i * 1024);
            if (lane < Ring::SB / 16) fb_dma(w.scales + at * Ring::SB, lane * 16, to + Ring::SCALES + i * Ring::SB);
            if constexpr (G > 0) {
                const uint8_t *z = w.zeros ? w.zeros + at * Ring::ZB : w.codes;
                if (lane < Ring::ZB / 16) fb_dma(z, lane * 16, to + Ring::ZEROS + i * Ring::ZB);
            }
        }
    };
    const int steps = wave < p.KT ? (p.KT - wave + WAVES - 1) / WAVES : 0;  // of this wave: wave, wave + WAVES, ...
    auto step = [&](int i) { return wave + WAVES * (i < steps ? i : 0); };   // (past the last: the first again, not multiplied)
    if (steps) {
#pragma unroll
        for (int i = 0; i < S - 1; ++i) issue(step(i), i);
    }
    if constexpr (G > 0) {
        if (tid < 16) tables[tid] = make_uint4(fb_table(tid, 0), fb_table(tid, 4), fb_table(tid, 8), fb_table(tid, 12));
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (not __syncthreads: that waits for the loads too)
    }
    const uint32_t zmask = p.w[0].zeros ? 0xffffffffu : 0u, znone = p.w[0].zeros ? 0u : 0x08080808u;
    f32x4_t acc[NT], a[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = f32x4_t{};
    constexpr int PER = G ? 4 / G : 1;  // matrix steps of a group
    const int xrow = lr & (4 * RX - 1);
    int slot = 0;
    for (int n = 0; n < steps; ++n) {
        // The slot that is filled next was read in the step before: those reads have returned (what they fed has been multiplied).
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        issue(step(n + S - 1), slot == 0 ? S - 1 : slot - 1);
        fb_wait<(S - 1) * Ring::LOADS>();
        const uint8_t *const st = ring + slot * Ring::BYTES;
        slot = slot == S - 1 ? 0 : slot + 1;
        uint4 c[NT], s[NT][G == 4 ? 2 : 1], x[4];
        uint32_t z[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if constexpr (G == 0) {
                z[i] = *reinterpret_cast<const uint32_t *>(st + Ring::SCALES + i * Ring::SB + lr * 4);
            } else {
                const uint8_t *zp = st + Ring::ZEROS + i * Ring::ZB + lr * G, *sp = st + Ring::SCALES + i * Ring::SB + kg * (8 * G);
                z[i] = G == 4 ? *reinterpret_cast<const uint32_t *>(zp) : G == 2 ? *reinterpret_cast<const uint16_t *>(zp) : *zp;
                z[i] = (z[i] & zmask) | znone;
                if constexpr (G == 1) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(sp);
                    s[i][0] = make_uint4(u.x, u.y, 0, 0);
                } else {
#pragma unroll
                    for (int g = 0; g < G / 2; ++g) s[i][g] = reinterpret_cast<const uint4 *>(sp)[g];
                }
            }
            c[i] = *reinterpret_cast<const uint4 *>(st + Ring::CODES + i * 1024 + lane * 16);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const uint4 *>(st + xrow * 256 + (((4 * j + kg) ^ xrow) << 4));
        uint4 tab[NT][G ? G : 1];
        if constexpr (G > 0) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int g = 0; g < G; ++g) tab[i][g] = tables[(z[i] >> (8 * g)) & 15u];
        }
        __builtin_amdgcn_sched_barrier(0);  // all reads are on their way before the first result is used
        const int left = p.K - 128 * step(n);  // of k: whole groups, a step but for the last
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (32 * j >= left) break;
            const bf16x8_t xv = __builtin_bit_cast(bf16x8_t, x[j]);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                if constexpr (G == 0) {
                    const bf16x8_t w = fb_e2m1(fb_word(c[i], j), mx_scale_operand((int)((z[i] >> (8 * j)) & 0xffu)));
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, xv, acc[i], 0, 0, 0);
                } else {
                    const int g = j / PER;
                    const bf16x8_t w = fb_int4(fb_word(c[i], j), tab[i][g]);
                    a[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, xv, j % PER ? a[i] : f32x4_t{}, 0, 0, 0);
                    if (j % PER == PER - 1) {
                        const uint32_t s0 = fb_word(s[i][g / 2], 2 * (g & 1)), s1 = fb_word(s[i][g / 2], 2 * (g & 1) + 1);
                        const float f[4] = {bf_lo(s0), bf_hi(s0), bf_lo(s1), bf_hi(s1)};
#pragma unroll
                        for (int v = 0; v < 4; ++v) acc[i][v] = __builtin_fmaf(f[v], a[i][v], acc[i][v]);
                    }
                }
            }
        }
    }
    fb_wait<0>();
    __syncthreads();
    f32x4_t(*const part)[NT][64] = reinterpret_cast<f32x4_t(*)[NT][64]>(lds);
#pragma unroll
    for (int i = 0; i < NT; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave >= OT) return;
    f32x4_t y = {}, u = {};
#pragma unroll
    for (int v = 0; v < WAVES; ++v) {
        y += part[v][SWIGLU ? 2 * wave : wave][lane];
        if (SWIGLU) u += part[v][2 * wave + 1][lane];
    }
    if (G) y *= 1.0f / FB_UNIT, u *= 1.0f / FB_UNIT;
    const int64_t n0 = ((int64_t)blockIdx.x * OT + wave) * 16 + 4 * kg;
    if (lr < 4 * RX && lr < rows && n0 < p.N) fb_store<SWIGLU>(p, row0 + lr, n0, y, u);
}

template <int G, int NT, int RX, int WAVES, int S, bool SWIGLU>
static int launch_fourbit_ring(const FourBitArgs &a, hipStream_t st) {
    constexpr int OT = SWIGLU ? NT / 2 : NT, bytes = FbRing<G, NT, RX, WAVES, S>::LDS;
    static std::atomic<bool> done[QIM_MAX_DEVICES];
    if (bytes > 65536) {
        const int rc = reserve_lds(reinterpret_cast<const void *>(k_fourbit<G, NT, RX, WAVES, S, SWIGLU>), bytes, done, "qim_fourbit_matmul");
        if (rc != QIM_OK) return rc;
    }
    launch(k_fourbit<G, NT, RX, WAVES, S, SWIGLU>, dim3((unsigned)(((a.N + 15) / 16 + OT - 1) / OT), (unsigned)((a.M + 4 * RX - 1) / (4 * RX))), dim3(64 * WAVES), bytes, st, a);
    return QIM_OK;
}

// More rows: a workgroup of WAVES = 8 or 4 waves and 16 NR x 64 or 32 values of output; of each step of 128 k, staged in LDS,
// wave w takes the k 32 (w % 4) .. + 31 for 32 of the columns, so that every code is made an operand once; or, in groups of 64
// or 128 k and up to 80 rows (KC 2), the k 64 (w % 2) .. + 63 for 16 columns: half of the scalings for twice the reads of x (300
// rows, 4096 -> 12288: 61.7 us and 52.1).  Two stages: one multiplied, one on its way (a third was slower: the step's chain of reads, operands and products holds it
// up); a stage's 16-byte chunk c of row r of x lies at c ^ (r % 16), so that the 16 rows of an operand lie in different banks.
template <int G, int NR, int WAVES>
struct FtStage {
    static constexpr int NT = WAVES / 2;  // 16-column tiles of W
    static constexpr int KC = (G == 1 || G == 2) && NR < 8 ? 2 : 1, KW = 4 / KC, TW = 2 / KC;  // a wave's steps of 32 k, waves along k, tiles a wave
    static constexpr int TP = KC == 1 ? 2 : NT;  // tiles joined at a time
    static constexpr int SB = G ? 32 * G : 64, ZB = 16 * G;  // bytes of a tile's scales or exponents, and of its zero points
    static constexpr int CODES = NR * 16 * 256, SCALES = CODES + NT * 1024, ZEROS = SCALES + NT * SB, BYTES = ZEROS + NT * ZB;
    static constexpr int JOIN = KW * TP * NR * 64 * 16;        // the waves' partial sums of those
    static constexpr int TABLES = 2 * BYTES > JOIN ? 2 * BYTES : JOIN, LDS = TABLES + (G ? 256 : 0);
};

template <int G, int NR, int WAVES, bool SWIGLU>
__global__ __launch_bounds__(64 * WAVES, 4) void k_fourbit_tile(FourBitArgs p, uint32_t ncol) {
    using St = FtStage<G, NR, WAVES>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    uint4 *const tables = reinterpret_cast<uint4 *>(lds + St::TABLES);
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    constexpr int KC = St::KC, TW = St::TW;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = KC * (wave % St::KW), part_of = wave / St::KW;  // first step of 32 k; of the columns
    const uint32_t rowblock = blockIdx.x / ncol, col = blockIdx.x - rowblock * ncol;
    const int row0 = (int)rowblock * 16 * NR;
    constexpr int OT = SWIGLU ? St::NT / 2 : St::NT;
    if constexpr (G > 0) {
        if (tid < 16) tables[tid] = make_uint4(fb_table(tid, 0), fb_table(tid, 4), fb_table(tid, 8), fb_table(tid, 12));
    }
    // This wave's part of a stage: 1 KiB pieces of x, 4 rows each, and of tile `of` of W the codes (the first NT waves) or the
    // scales and zero points (the others).  Rows and tiles past the last are the last, and of k past the end others come: nothing
    // multiplies with them.
    const int ntiles = (p.N + 15) / 16, of = wave % St::NT, mine = (int)col * OT + (SWIGLU ? of >> 1 : of);
    const FourBitWeight &fw = p.w[SWIGLU ? of & 1 : 0];
    const int64_t tile = mine < ntiles ? mine : ntiles - 1;
    const uint8_t *const x0 = reinterpret_cast<const uint8_t *>(p.x + row0 * p.ldx);
    const uint8_t *const wc = fw.codes + tile * p.KT * 1024, *const ws = fw.scales + tile * p.KT * St::SB;
    const uint8_t *const wz = G && fw.zeros ? fw.zeros + tile * p.KT * St::ZB : wc;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)lds;
    constexpr int PIECES = (4 * NR + WAVES - 1) / WAVES;
    uint32_t xoff[PIECES];
    auto piece = [&](int i) { return (wave + WAVES * i) % (4 * NR); };  // (some come twice, where 2 does not divide NR)
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int r = 4 * piece(i) + kg, last = p.M - 1 - row0;
        xoff[i] = (uint32_t)(r < last ? r : last) * (uint32_t)(2 * p.ldx) + 16 * (lr ^ (r & 15));
    }
    auto issue = [&](int t, int slot) {
        const uint32_t to = lds0 + slot * St::BYTES;
        const uint8_t *const xt = x0 + (int64_t)t * 256;
        const bool whole = 128 * t + 128 <= p.K;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            uint32_t off = xoff[i];
            if (!whole) {
                const int k = 8 * (lr ^ ((4 * piece(i) + kg) & 15));
                off -= 128 * t + k < p.K ? 0 : 2 * k;
            }
            fb_dma(xt, off, to + piece(i) * 1024);
        }
        if (wave < St::NT) {
            fb_dma(wc + (int64_t)t * 1024, lane * 16, to + St::CODES + of * 1024);
        } else {
            if (lane < St::SB / 16) fb_dma(ws + (int64_t)t * St::SB, lane * 16, to + St::SCALES + of * St::SB);
            if constexpr (G > 0) {
                if (lane < St::ZB / 16) fb_dma(wz + (int64_t)t * St::ZB, lane * 16, to + St::ZEROS + of * St::ZB);
            }
        }
    };

    f32x4_t acc[TW][NR];
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[i][r] = f32x4_t{};
    const int g = G ? j * G / 4 : 0;  // the group of this wave's k
    const uint32_t zmask = fw.zeros ? 15u : 0u, znone = fw.zeros ? 0u : 8u;
    issue(0, 0);
    for (int t = 0; t < p.KT; ++t) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the stage is there, the other has been read
        if (t + 1 < p.KT) issue(t + 1, (t + 1) & 1);
        const uint8_t *const st = lds + (t & 1) * St::BYTES;
        if (128 * t + 32 * j < p.K) {
            uint32_t c[TW][KC];
            uint2 s2[TW];
            uint4 tab[TW];
            uint32_t e[TW];
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                const int n = TW * part_of + i;
                const uint8_t *const cp = st + St::CODES + n * 1024 + lane * 16 + 4 * j;
                if constexpr (KC == 2) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(cp);
                    c[i][0] = u.x, c[i][1] = u.y;
                } else {
                    c[i][0] = *reinterpret_cast<const uint32_t *>(cp);
                }
                if constexpr (G == 0) {
                    e[i] = st[St::SCALES + n * St::SB + lr * 4 + j];
                } else {
                    s2[i] = *reinterpret_cast<const uint2 *>(st + St::SCALES + n * St::SB + (kg * G + g) * 8);
                    tab[i] = tables[(st[St::ZEROS + n * St::ZB + lr * G + g] & zmask) | znone];
                }
            }
            bf16x8_t x[KC][NR];
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int r = 0; r < NR; ++r) x[k][r] = *reinterpret_cast<const bf16x8_t *>(st + (16 * r + lr) * 256 + (((4 * (j + k) + kg) ^ lr) << 4));
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                if constexpr (G == 0) {
                    const bf16x8_t w = fb_e2m1(c[i][0], mx_scale_operand((int)e[i]));
#pragma unroll
                    for (int r = 0; r < NR; ++r) acc[i][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[0][r], acc[i][r], 0, 0, 0);
                } else {
                    const float s[4] = {bf_lo(s2[i].x), bf_hi(s2[i].x), bf_lo(s2[i].y), bf_hi(s2[i].y)};
                    bf16x8_t w[KC];
#pragma unroll
                    for (int k = 0; k < KC; ++k) w[k] = fb_int4(c[i][k], tab[i]);
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        f32x4_t a = f32x4_t{};
#pragma unroll
                        for (int k = 0; k < KC; ++k) a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[k], x[k][r], a, 0, 0, 0);
#pragma unroll
                        for (int n = 0; n < 4; ++n) acc[i][r][n] = __builtin_fmaf(s[n], a[n], acc[i][r][n]);
                    }
                }
            }
        }
    }
    // The join, TP tiles at a time.
    constexpr int TP = St::TP;
    f32x4_t(*const part)[TP * NR][64] = reinterpret_cast<f32x4_t(*)[TP * NR][64]>(lds);
#pragma unroll
    for (int h = 0; h < St::NT / TP; ++h) {
        __syncthreads();
        if (part_of * TW / TP == h) {
#pragma unroll
            for (int i = 0; i < TW; ++i)
#pragma unroll
                for (int r = 0; r < NR; ++r) part[wave % St::KW][(part_of * TW % TP + i) * NR + r][lane] = acc[i][r];
        }
        __syncthreads();
        constexpr int OP = SWIGLU ? TP / 2 : TP, BLOCKS = OP * NR;
#pragma unroll
        for (int i = 0; i < (BLOCKS + WAVES - 1) / WAVES; ++i) {
            const int blk = wave + WAVES * i, ot = blk / NR, r = blk - ot * NR, first = (SWIGLU ? 2 * ot : ot) * NR + r;
            if (blk >= BLOCKS) break;
            f32x4_t y = {}, u = {};
#pragma unroll
            for (int v = 0; v < St::KW; ++v) {
                y += part[v][first][lane];
                if (SWIGLU) u += part[v][first + NR][lane];
            }
            if (G) y *= 1.0f / FB_UNIT, u *= 1.0f / FB_UNIT;
            const int64_t n0 = ((int64_t)col * OT + h * OP + ot) * 16 + 4 * kg;
            const int row = row0 + 16 * r + lr;
            if (row < p.M && n0 < p.N) fb_store<SWIGLU>(p, row, n0, y, u);
        }
    }
}

template <int G, int NR, int WAVES, bool SWIGLU>
static int launch_fourbit_tile(const FourBitArgs &a, hipStream_t st) {
    using St = FtStage<G, NR, WAVES>;
    constexpr int OT = SWIGLU ? St::NT / 2 : St::NT, bytes = St::LDS;
    const uint32_t ncol = (uint32_t)(((a.N + 15) / 16 + OT - 1) / OT);
    const int64_t wgs = (int64_t)ncol * ((a.M + 16 * NR - 1) / (16 * NR));
    QIM_REQUIRE(wgs * (64 * WAVES) < (1ll << 32), QIM_ERR_SHAPE, "qim_fourbit_matmul: M %d, N %d: too large", a.M, a.N);
    static std::atomic<bool> done[QIM_MAX_DEVICES];
    if (bytes > 65536) {
        const int rc = reserve_lds(reinterpret_cast<const void *>(k_fourbit_tile<G, NR, WAVES, SWIGLU>), bytes, done, "qim_fourbit_matmul");
        if (rc != QIM_OK) return rc;
    }
    launch(k_fourbit_tile<G, NR, WAVES, SWIGLU>, dim3((unsigned)wgs), dim3(64 * WAVES), bytes, st, a, ncol);
    return QIM_OK;
}

// Which kernel.  At 4096 columns of x (where the times were taken; other widths choose alike) the tile kernel takes about 3.5 + 2.75 NR us for each workgroup of
// eight waves that a CU has to take (groups of 64 and 128, up to 80 rows: 4 + 2.2 NR), a third more where it takes one only,
// and up to 10 us besides; the ring kernel 1.5 us and 2.75 for each of the CU's tiles of 16 x 16.  The first is held up by the
// chain of its steps while a CU has few workgroups, the other makes operands of all codes again for every 16 rows.
// int4, group 64, tile against ring: 32 x 4096 18.2 us and 9.7, 64 x 4096 18.3 and 12.7, 128 x 4096 16.7 and 21.7, 24 x 24576
// 21.1 and 33.1, 16 x 65536 41.7 and 48.2; mxfp4: 64 x 4096 17.1 and 8.9, 16 x 65536 31.7 and 39.0.  Tiles of 64 rows
// against 128, group 64: 512 x 4096 31.3 us and 38.5, 1024 x 4096 58.5 and 56.4.
// Up to one and a half workgroups of eight waves a CU int4 takes workgroups of four instead, which divide the CUs more evenly and
// wait for fewer at a barrier (us, eight waves and four: 24 x 12288 SwiGLU 26.6, 23.8; 154 x 12288, group 32, 39.8, 35.1; 128 x
// 4096 20.3, 18.0; but 300 x 12288, three a CU, 60.9 and 67.4, and mxfp4 154 x 12288 24.4 and 25.5).
template <int G, bool SWIGLU>
static int launch_fourbit(const FourBitArgs &a, hipStream_t st) {
    constexpr int ONE = SWIGLU ? 2 : 1, OT = 4 / ONE;
    if (a.M <= 4) return launch_fourbit_ring<G, ONE, 1, 8, 3, SWIGLU>(a, st);
    const int64_t ntiles = (a.N + 15) / 16, ncol = (ntiles + OT - 1) / OT;
    auto wgs = [&](int nr) { return ncol * ((a.M + 16 * nr - 1) / (16 * nr)); };  // of eight waves
    auto four = [&](int nr) { return G > 0 && nr > 1 && nr < 8 && wgs(nr) <= 384; };
    constexpr bool wide = G == 1 || G == 2;  // (FtStage's KC 2)
    auto cost = [&](int nr) {  // of 0.0275 us
        const int64_t n = wgs(nr);
        return (n <= 256 ? four(nr) ? 11 : 13 : four(nr) ? 15 : (n + 255) / 256 * 10) * (wide && nr < 8 ? 8 * nr + 16 : 10 * nr + 13);
    };
    int nr = 8;
    for (int n : {5, 4, 2, 1})
        if (cost(n) < cost(nr)) nr = n;
    const int64_t blocks = (a.M + 15) / 16 * ntiles;
    if (a.M <= 16 * 65535 && 100 * ONE * blocks < 256 * ((wide ? 190 : 350) + cost(nr))) {  // (a grid of no more than 65535 blocks of rows)
        // From one and a half tiles a CU on two of them share the reads of x, and two workgroups of four waves a CU take more of
        // them at a time (16 rows, mxfp4: 4096 -> 12288 9.2 us against 11.6; 12288 -> 4096, 256 tiles, 14.6 against 9.0).
        if (blocks >= 384) return launch_fourbit_ring<G, 2, 4, 4, 3, SWIGLU>(a, st);
        return launch_fourbit_ring<G, ONE, 4, 8, 2, SWIGLU>(a, st);
    }
    if constexpr (G > 0) {
        if (four(nr)) {
            switch (nr) {
                case 2: return launch_fourbit_tile<G, 2, 4, SWIGLU>(a, st);
                case 4: return launch_fourbit_tile<G, 4, 4, SWIGLU>(a, st);
                default: return launch_fourbit_tile<G, 5, 4, SWIGLU>(a, st);
            }
        }
    }
    switch (nr) {
        case 1: return launch_fourbit_tile<G, 1, 8, SWIGLU>(a, st);
        case 2: return launch_fourbit_tile<G, 2, 8, SWIGLU>(a, st);
        case 4: return launch_fourbit_tile<G, 4, 8, SWIGLU>(a, st);
        case 5: return launch_fourbit_tile<G, 5, 8, SWIGLU>(a, st);
        default: return launch_fourbit_tile<G, 8, 8, SWIGLU>(a, st);
    }
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
    QIM_REQUIRE(ldx >= K && ldx % 8 == 0 && ldx < (1 << 24) && ldo >= N && aligned16(x) && aligned16(codes) && aligned16(scales) && aligned16(zeros) &&
                    aligned16(codes2) && aligned16(scales2) && aligned16(zeros2) &&
                    (reinterpret_cast<uintptr_t>(out) & (out_f32 ? 3u : 1u)) == 0 && (reinterpret_cast<uintptr_t>(bias) & 1u) == 0,
                QIM_ERR_LAYOUT, "%s: rows of x must be 16-byte aligned and fewer than 2^24 elements apart", who);
    const int64_t size = out_f32 ? 4 : 2;
    QIM_REQUIRE(!bytes_share(out, size * ((M - 1) * ldo + N), x, 2 * ((M - 1) * ldx + K)), QIM_ERR_ARG, "%s: out overlaps x", who);
    // (codes, scales or exponents, zero points: of 16 rows and 128 k)
    const int64_t steps = (N + 15) / 16 * ((K + 127) / 128), per = group ? 128 / group : 0;
    const struct {
        const void *at;
        int64_t bytes;
    } inputs[] = {{codes, 1024 * steps}, {codes2, 1024 * steps}, {scales, (group ? 32 * per : 64) * steps}, {scales2, (group ? 32 * per : 64) * steps},
                  {zeros, 16 * per * steps}, {zeros2, 16 * per * steps}, {bias, 2 * N}};
    for (const auto &in : inputs)
        QIM_REQUIRE(!rows_share_vectors(out, ldo * size / 2, N * size / 2, M, in.at, 0, 1, in.bytes / 2), QIM_ERR_ARG,
                    "%s: out overlaps a weight or the bias", who);
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
