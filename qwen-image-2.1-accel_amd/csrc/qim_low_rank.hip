// Low-rank adapters of several requests beside one shared projection:
//
//   out[m] = base[m] + scale[a] * up[a] (down[a] x[m]),   a = index[m / seq]
//
// in two launches (in one for a few short rows, k_lr_small).  k_lr_down: h = down x,
// (M, parts * R) in fp32, with the K axis cut into chunks where there are few rows
// (each chunk's sums go to the workspace).  k_lr_up: adds the chunks, multiplies by up
// and adds to base.
//
// Both products have their long operand's rows as MFMA columns
// (v_mfma_f32_16x16x32_bf16, D = A B with A = the adapter's rows and B = rows of
// x or h), so a lane owns one row m of the batch in the result.  Rows of one
// 16-row tile may belong to different adapters: the tile's distinct adapters
// are taken in turn over the same rows, and a lane keeps the result of its
// own row's adapter.  Nothing is masked by multiplying, so a request's infinities or
// NaN stay in its own rows.
//
// h stays fp32 between the launches and enters the second product as two bf16
// terms, h = hi + lo (lo the rounding error of hi): 16 significand bits where one
// bf16 would put 2^-9 of each term into the sum.  The second term costs matrix
// cycles, which these launches have to spare: they move x, base and out once
// and are bound by that.  8192 rows, K 4096, N 12288 in 3 parts of rank 16, 2 adapters:
// down 29 us (67 MB of x; ~9 of it are start and join), up 88 us (402 MB, 4.6 TB/s).
// 2381 rows of mixed adapters, K 12288, N 4096, rank 64: 25 and 21 us; a second
// adapter of a row tile costs 3-4 us (its x comes from L2), less than ordering the
// rows by adapter first (7 us and scattered rows).
#include "qim_device.h"
#include "qim_runtime.h"

namespace qim {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct LowRankArgs {
    const uint16_t *x, *down, *up, *base;
    const int32_t *index;
    const float *scale;
    uint16_t *out;
    float *h;  // (chunks, M, PR)
    int64_t ldx, ldb, ldo, M;
    uint32_t seq;
    int K, N, R, PR, parts, A;
    int chunks, kchunk;  // K chunks of kchunk values
    int ncols, nchunk;   // k_lr_up: columns of a part per wave; workgroups per part
};

// The adapter of row m, -1 for none.
__device__ __forceinline__ int lr_adapter(const LowRankArgs &p, int64_t m) {
    if (m >= p.M) return -1;
    const int a = p.index[p.seq == 1 ? (uint32_t)m : (uint32_t)m / p.seq];
    return a >= 0 && a < p.A ? a : -1;
}

// Calls f(a) for each distinct adapter a >= 0 among the rows of MT tiles whose
// rank in that order is `slot` modulo `slots`.
template <int MT, class F>
__device__ __forceinline__ void lr_each(const int (&mine)[MT], int slot, int slots, F &&f) {
    uint64_t todo[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) todo[t] = __builtin_amdgcn_ballot_w64(mine[t] >= 0);
    int rank = slot;
    for (;;) {
        int a = -1;
#pragma unroll
        for (int t = 0; t < MT; ++t)
            if (a < 0 && todo[t]) a = __builtin_amdgcn_readlane(mine[t], (int)__builtin_ctzll(todo[t]));
        if (a < 0) return;
#pragma unroll
        for (int t = 0; t < MT; ++t) todo[t] &= ~__builtin_amdgcn_ballot_w64(mine[t] == a);
        if (rank == 0) f(a);
        rank = rank == 0 ? slots - 1 : rank - 1;
    }
}

// h of 16 * MT rows, one K chunk and 16 * RT rows of down.  The 8 waves take
// steps of 32 * S values of the chunk in turn (S = 2: whole 128-byte lines of x;
// 1 where RT = 8 leaves no registers), with the next step's loads in flight,
// and join in LDS.
constexpr int LR_WAVES = 8;
template <int RT, int MT>
__global__ __launch_bounds__(64 * LR_WAVES, 2) void k_lr_down(LowRankArgs p, int rblocks) {
    constexpr int S = RT == 8 ? 1 : 2;
    extern __shared__ f32x4_t sum[];  // [LR_WAVES][MT][RT][64]
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Neighbouring workgroups take neighbouring chunks of the same rows: what is
    // in flight covers whole rows.
    const uint32_t tile = blockIdx.x / (uint32_t)p.chunks, chunk = blockIdx.x - tile * p.chunks;
    const int64_t m0 = (int64_t)tile * (16 * MT);
    const int slot = blockIdx.y / rblocks, slots = gridDim.y / rblocks, r0 = (blockIdx.y - slot * rblocks) * (16 * RT);
    int mine[MT];
    const uint16_t *xr[MT];
    uint64_t done[MT];  // the lanes whose rows this workgroup computes
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t m = m0 + 16 * t + lr;
        mine[t] = lr_adapter(p, m);
        xr[t] = p.x + (m < p.M ? m : p.M - 1) * p.ldx + 8 * kg;
        done[t] = 0;
    }
    const int k0 = chunk * p.kchunk, k1 = k0 + p.kchunk < p.K ? k0 + p.kchunk : p.K;
    lr_each<MT>(mine, slot, slots, [&](int a) {
        const uint16_t *dn[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            int row = r0 + 16 * r + lr;
            row = row < p.PR ? row : p.PR - 1;
            dn[r] = p.down + ((int64_t)a * p.PR + row) * p.K + 8 * kg;
        }
        f32x4_t acc[MT][RT];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[t][r] = f32x4_t{};
        u32x4_t xc[MT][S], dc[RT][S], xn[MT][S], dnx[RT][S];
        auto load = [&](int k, u32x4_t (&xv)[MT][S], u32x4_t (&dv)[RT][S]) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const bool in = k + 32 * s + 8 * kg < k1;  // K % 8 == 0: 8 values are all in or all out
                const u32x4_t zero = {0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < MT; ++t) xv[t][s] = in ? *reinterpret_cast<const u32x4_t *>(xr[t] + k + 32 * s) : zero;
#pragma unroll
                for (int r = 0; r < RT; ++r) dv[r][s] = in ? *reinterpret_cast<const u32x4_t *>(dn[r] + k + 32 * s) : zero;
            }
        };
        int k = k0 + 32 * S * wave;
        load(k, xc, dc);
        for (; k < k1; k += 32 * S * LR_WAVES) {
            if (k + 32 * S * LR_WAVES < k1) load(k + 32 * S * LR_WAVES, xn, dnx);
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
                        acc[t][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, dc[r][s]),
                                                                            __builtin_bit_cast(bf16x8_t, xc[t][s]), acc[t][r], 0, 0, 0);
#pragma unroll
            for (int s = 0; s < S; ++s) {
#pragma unroll
                for (int t = 0; t < MT; ++t) xc[t][s] = xn[t][s];
#pragma unroll
                for (int r = 0; r < RT; ++r) dc[r][s] = dnx[r][s];
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            done[t] |= __builtin_amdgcn_ballot_w64(mine[t] == a);
            if (mine[t] == a) {
#pragma unroll
                for (int r = 0; r < RT; ++r) sum[((wave * MT + t) * RT + r) * 64 + lane] = acc[t][r];
            }
        }
    });
    __syncthreads();
    for (int i = tid; i < MT * RT * 64; i += 64 * LR_WAVES) {
        const int t = i / (RT * 64), r = (i >> 6) % RT, l = i & 63;
        f32x4_t s = sum[i];
#pragma unroll
        for (int w = 1; w < LR_WAVES; ++w) s += sum[w * (MT * RT * 64) + i];
        // Lane l of the tile: row l % 16, values 4 (l / 16) .. + 3 of its 16.
        const int row = 16 * t + (l & 15), col = r0 + 16 * r + 4 * (l >> 4);
        uint64_t rows = done[0];
#pragma unroll
        for (int u = 1; u < MT; ++u) rows = t == u ? done[u] : rows;
        if (((rows >> l) & 1) && col < p.PR)
            *reinterpret_cast<f32x4_t *>(p.h + ((int64_t)chunk * p.M + m0 + row) * p.PR + col) = s;
    }
}

// 32 rows x 4 * ncols columns of one part: the workgroup sums the K chunks of its
// rows' h once, into LDS, as MFMA operands; each wave takes 64 columns at a
// time, with its next 64 columns of base in flight.  SP =
// ceil(R / 32) operand steps of hi and as many of lo; with PACK (R <= 16) one step holds
// both (slots of 8: hi, hi, lo, lo).  A tile's 16 result rows are assigned to
// columns so that a lane's results of two tiles are 8 neighbouring
// columns: row i of tile t of a pair is column 8 (i / 4) + 4 t + i % 4.
constexpr int LR_MT = 2;
template <int SP, bool PACK>
__global__ __launch_bounds__(256, SP == 4 ? 2 : 3) void k_lr_up(LowRankArgs p) {
    constexpr int OPS = PACK ? 1 : 2 * SP;
    __shared__ u32x4_t hs[LR_MT][OPS][64];
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Neighbouring workgroups take neighbouring columns of the same rows, and the
    // four waves neighbouring 64-column steps: what is in flight covers whole rows.
    const uint32_t cols = (uint32_t)(p.nchunk * p.parts), tile = blockIdx.x / cols, cb = blockIdx.x - tile * cols;
    const int64_t m0 = (int64_t)tile * (16 * LR_MT);
    const int part = cb / p.nchunk, width = p.N / p.parts;
    const int rc = p.R / 8;  // chunks of 8
    const int g0 = (cb - part * p.nchunk) * 4 * p.ncols;
    const int c0 = g0 + 64 * wave, c1 = g0 + 4 * p.ncols < width ? g0 + 4 * p.ncols : width;
    const int64_t n0 = (int64_t)part * width;
    // Base columns c .. c + 63.
    auto load_base = [&](int c, uint4 (&y)[LR_MT][2]) {
#pragma unroll
        for (int t = 0; t < LR_MT; ++t)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int64_t m = m0 + 16 * t + lr;
                const int col = c + 32 * g + 8 * kg;
                y[t][g] = make_uint4(0, 0, 0, 0);
                if (p.base && m < p.M && col < c1) y[t][g] = *reinterpret_cast<const uint4 *>(p.base + m * p.ldb + n0 + col);
            }
    };
    int mine[LR_MT];
#pragma unroll
    for (int t = 0; t < LR_MT; ++t) mine[t] = lr_adapter(p, m0 + 16 * t + lr);
    uint4 yc[LR_MT][2];
    load_base(c0, yc);  // in flight while h is fetched
    bool again = false;
    // h of the workgroup's rows.
    for (int i = tid; i < LR_MT * SP * 64; i += 256) {
        const int t = i / (SP * 64), s = (i >> 6) % SP, l = i & 63;
        const int64_t m = m0 + 16 * t + (l & 15);
        const int ch = PACK ? (l >> 4) & 1 : 4 * s + (l >> 4);
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, lo[8];
        if (ch < rc && m < p.M) {  // of a row without an adapter: never written, and its results are not used
            const float *src = p.h + m * p.PR + part * p.R + ch * 8;
            for (int c = 0; c < p.chunks; c += 4) {  // four chunks' loads at a time
                f32x4_t a[4], b[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4_t *at = reinterpret_cast<const f32x4_t *>(src + (c + j < p.chunks ? j : 0) * p.M * p.PR);
                    a[j] = at[0];
                    b[j] = at[1];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f[e] += c + j < p.chunks ? a[j][e] : 0.f;
                        f[4 + e] += c + j < p.chunks ? b[j][e] : 0.f;
                    }
                src += 4 * p.M * p.PR;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float hi = rbf(f[e]);
            lo[e] = __builtin_isfinite(hi) ? f[e] - hi : 0.0f;
        }
        const uint4 uh = pack8(f), ul = pack8(lo);
        const u32x4_t vh = {uh.x, uh.y, uh.z, uh.w}, vl = {ul.x, ul.y, ul.z, ul.w};
        if (PACK) {
            hs[t][0][l] = l < 32 ? vh : vl;
        } else {
            hs[t][s][l] = vh;
            hs[t][OPS / 2 + s][l] = vl;
        }
    }
    __syncthreads();
    bf16x8_t hop[LR_MT][OPS];
#pragma unroll
    for (int t = 0; t < LR_MT; ++t)
#pragma unroll
        for (int s = 0; s < OPS; ++s) hop[t][s] = __builtin_bit_cast(bf16x8_t, hs[t][s][lane]);

    auto store = [&](int a, int c, int t, int g, const uint4 &y) {
        const int64_t m = m0 + 16 * t + lr;
        const int col = c + 32 * g + 8 * kg;
        if (mine[t] == a && m < p.M && col < c1) *reinterpret_cast<uint4 *>(p.out + m * p.ldo + n0 + col) = y;
    };
    if (blockIdx.y == 0 && p.base != p.out) {  // rows without an adapter: copied
        bool none = false;
#pragma unroll
        for (int t = 0; t < LR_MT; ++t) none |= mine[t] < 0 && m0 + 16 * t + lr < p.M;
        if (__builtin_amdgcn_ballot_w64(none)) {
            for (int c = c0; c < c1; c += 256) {
                uint4 y[LR_MT][2];
                load_base(c, y);
#pragma unroll
                for (int t = 0; t < LR_MT; ++t)
#pragma unroll
                    for (int g = 0; g < 2; ++g) store(-1, c, t, g, y[t][g]);
            }
        }
    }
    lr_each<LR_MT>(mine, blockIdx.y, gridDim.y, [&](int a) {
        const float sc = p.scale ? p.scale[a] : 1.0f;
        const uint16_t *up = p.up + ((int64_t)a * p.N + n0) * p.R;
        uint4 yn[LR_MT][2];
        if (again) load_base(c0, yc);
        again = true;
        u32x4_t uc[4][SP], un[4][SP];
        auto load_up = [&](int c, u32x4_t (&u)[4][SP]) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                int n = c + 32 * (q >> 1) + 8 * (lr >> 2) + 4 * (q & 1) + (lr & 3);
                n = n < width ? n : width - 1;
                const uint16_t *row = up + (int64_t)n * p.R;
#pragma unroll
                for (int s = 0; s < SP; ++s) {
                    const int ch = PACK ? kg & 1 : 4 * s + kg;
                    const u32x4_t zero = {0, 0, 0, 0};
                    u[q][s] = ch < rc ? *reinterpret_cast<const u32x4_t *>(row + ch * 8) : zero;
                }
            }
        };
        constexpr bool AHEAD = SP == 1;  // the next columns' operands too, where registers allow
        if (AHEAD) load_up(c0, uc);
        for (int c = c0; c < c1; c += 256) {
            if (!AHEAD) load_up(c, uc);
            if (c + 256 < c1) {
                load_base(c + 256, yn);
                if (AHEAD) load_up(c + 256, un);
            }
            f32x4_t acc[LR_MT][4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int t = 0; t < LR_MT; ++t) {
                    acc[t][q] = f32x4_t{};
#pragma unroll
                    for (int s = 0; s < SP; ++s) {
                        const bf16x8_t u = __builtin_bit_cast(bf16x8_t, uc[q][s]);
                        acc[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u, hop[t][s], acc[t][q], 0, 0, 0);
                        if (!PACK) acc[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u, hop[t][OPS / 2 + s], acc[t][q], 0, 0, 0);
                    }
                }
#pragma unroll
            for (int t = 0; t < LR_MT; ++t)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    float y[8];
                    unpack8(yc[t][g], y);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[e] = __builtin_fmaf(sc, acc[t][2 * g][e], y[e]);
                        y[4 + e] = __builtin_fmaf(sc, acc[t][2 * g + 1][e], y[4 + e]);
                    }
                    store(a, c, t, g, pack8(y));
                }
#pragma unroll
            for (int t = 0; t < LR_MT; ++t)
#pragma unroll
                for (int g = 0; g < 2; ++g) yc[t][g] = yn[t][g];
            if (AHEAD) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int s = 0; s < SP; ++s) uc[q][s] = un[q][s];
            }
        }
    });
}

// At most 16 rows of few values each: both products in one launch.  A workgroup
// takes 8 * 64 columns of one part for the adapters of its slot, and computes
// h for them itself: it reads R rows of down (again in every workgroup of that
// adapter, from L2) and the x of the adapter's own rows, the 8 waves taking
// steps of 128 values in turn, joins h in LDS, and multiplies by its columns of up.
// SP, PACK and the operands are k_lr_up's.
template <int SP, bool PACK>
__global__ __launch_bounds__(512, 2) void k_lr_small(LowRankArgs p) {
    constexpr int RT = PACK ? 1 : 2 * SP;  // 16-row tiles of down
    __shared__ f32x4_t sum[8][RT][64];
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int part = blockIdx.x / p.nchunk, width = p.N / p.parts, rc = p.R / 8;
    const int c = (blockIdx.x - part * p.nchunk) * 512 + 64 * wave;
    const int64_t n0 = (int64_t)part * width;
    const bool row = lr < p.M;
    uint4 y[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int col = c + 32 * g + 8 * kg;
        if (p.base && row && col < width) y[g] = *reinterpret_cast<const uint4 *>(p.base + lr * p.ldb + n0 + col);
    }
    const int mine[1] = {lr_adapter(p, lr)};
    if (blockIdx.y == 0 && p.base != p.out && mine[0] < 0 && row) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int col = c + 32 * g + 8 * kg;
            if (col < width) *reinterpret_cast<uint4 *>(p.out + lr * p.ldo + n0 + col) = y[g];
        }
    }
    lr_each<1>(mine, blockIdx.y, gridDim.y, [&](int a) {
        const bool own = mine[0] == a;
        const uint16_t *xr = p.x + (own ? lr : 0) * p.ldx + 8 * kg, *dn[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int at = 16 * r + lr < p.R ? 16 * r + lr : p.R - 1;
            dn[r] = p.down + ((int64_t)a * p.PR + part * p.R + at) * p.K + 8 * kg;
        }
        f32x4_t acc[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[r] = f32x4_t{};
        constexpr int S = PACK ? 4 : 2;  // 32-value steps whose loads go together
        u32x4_t xc[S], dc[RT][S], xn[S], dx[RT][S];
        auto load = [&](int k, u32x4_t (&xv)[S], u32x4_t (&dv)[RT][S]) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const bool in = k + 32 * s + 8 * kg < p.K;
                const u32x4_t zero = {0, 0, 0, 0};
                xv[s] = in && own ? *reinterpret_cast<const u32x4_t *>(xr + k + 32 * s) : zero;
#pragma unroll
                for (int r = 0; r < RT; ++r) dv[r][s] = in ? *reinterpret_cast<const u32x4_t *>(dn[r] + k + 32 * s) : zero;
            }
        };
        int k = 32 * S * wave;
        load(k, xc, dc);
        for (; k < p.K; k += 256 * S) {
            if (k + 256 * S < p.K) load(k + 256 * S, xn, dx);
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, dc[r][s]),
                                                                     __builtin_bit_cast(bf16x8_t, xc[s]), acc[r], 0, 0, 0);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                xc[s] = xn[s];
#pragma unroll
                for (int r = 0; r < RT; ++r) dc[r][s] = dx[r][s];
            }
        }
        // up of this wave's columns, in flight over the join.
        u32x4_t up[4][SP];
        const uint16_t *ua = p.up + ((int64_t)a * p.N + n0) * p.R;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            int n = c + 32 * (q >> 1) + 8 * (lr >> 2) + 4 * (q & 1) + (lr & 3);
            n = n < width ? n : width - 1;
#pragma unroll
            for (int s = 0; s < SP; ++s) {
                const int ch = PACK ? kg & 1 : 4 * s + kg;
                const u32x4_t zero = {0, 0, 0, 0};
                up[q][s] = ch < rc ? *reinterpret_cast<const u32x4_t *>(ua + (int64_t)n * p.R + ch * 8) : zero;
            }
        }
        __syncthreads();  // the previous adapter's sums have been read
#pragma unroll
        for (int r = 0; r < RT; ++r) sum[wave][r][lane] = acc[r];
        __syncthreads();
        f32x4_t res[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) res[q] = f32x4_t{};
#pragma unroll
        for (int s = 0; s < SP; ++s) {
            // Chunk ch of row lr: two lanes' values of tile ch / 2.
            const int ch = PACK ? kg & 1 : 4 * s + kg, at = (ch & 1) * 32 + lr;
            float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, hi[8], lo[8];
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                const f32x4_t u = sum[w][ch >> 1][at], v = sum[w][ch >> 1][at + 16];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f[e] += u[e];
                    f[4 + e] += v[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = ch < rc ? f[e] : 0.f;
                hi[e] = rbf(f[e]);
                lo[e] = __builtin_isfinite(hi[e]) ? f[e] - hi[e] : 0.f;
                if (PACK && kg >= 2) hi[e] = lo[e];
            }
            const bf16x8_t h0 = __builtin_bit_cast(bf16x8_t, pack8(hi)), h1 = __builtin_bit_cast(bf16x8_t, pack8(lo));
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const bf16x8_t u = __builtin_bit_cast(bf16x8_t, up[q][s]);
                res[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u, h0, res[q], 0, 0, 0);
                if (!PACK) res[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u, h1, res[q], 0, 0, 0);
            }
        }
        const float sc = p.scale ? p.scale[a] : 1.0f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int col = c + 32 * g + 8 * kg;
            float f[8];
            unpack8(y[g], f);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[e] = __builtin_fmaf(sc, res[2 * g][e], f[e]);
                f[4 + e] = __builtin_fmaf(sc, res[2 * g + 1][e], f[4 + e]);
            }
            if (own && col < width) *reinterpret_cast<uint4 *>(p.out + lr * p.ldo + n0 + col) = pack8(f);
        }
    });
}

// The launches' shapes.  Row tiles of the first: 64 rows (32 where R is large:
// registers, or where R and M are small: fewer, longer chunks), 16 for at most 16 rows.
// K chunks: as many as still fit one round of a workgroup per CU, each with
// at least 512 values (a step per wave).  Slots: where that is still too few,
// the distinct adapters of a row tile (at most `distinct` of them) go to
// different workgroups.
struct LrPlan {
    int rt, mt, ncols;
    int64_t rblocks, tiles, chunks, kchunk, slots, nchunk, up_slots;
};
static LrPlan lr_plan(int64_t M, int64_t seq, int64_t K, int64_t PR, int64_t width, int64_t parts, int64_t A) {
    const int64_t cus = device_cus() > 0 ? device_cus() : 256;
    auto upto = [](int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; };
    auto distinct = [&](int64_t rows) {
        const int64_t n = seq % rows == 0 ? 1 : (rows < M ? rows : M) / seq + (seq > 1 ? 2 : 0);
        return upto(n < A ? n : A, 1, 64);
    };
    LrPlan pl;
    pl.rt = PR <= 16 ? 1 : PR <= 32 ? 2 : PR <= 64 ? 4 : 8;
    pl.mt = M <= 16 ? 1 : pl.rt == 8 || (pl.rt <= 2 && M < 32 * cus) ? 2 : 4;
    pl.rblocks = (PR + 16 * pl.rt - 1) / (16 * pl.rt);
    pl.tiles = (M + 16 * pl.mt - 1) / (16 * pl.mt);
    constexpr int64_t step = 64 * LR_WAVES;
    const int64_t chunks = upto(cus / (pl.tiles * pl.rblocks), 1, upto((K + step - 1) / step, 1, 16));
    pl.kchunk = ((K + chunks - 1) / chunks + step - 1) / step * step;
    pl.chunks = (K + pl.kchunk - 1) / pl.kchunk;  // none empty after rounding
    pl.slots = upto(upto(cus / (pl.tiles * pl.rblocks * pl.chunks), 2, 64), 1, distinct(16 * pl.mt));
    const int64_t up_tiles = (M + 16 * LR_MT - 1) / (16 * LR_MT);
    pl.ncols = 256;
    for (; pl.ncols > 64 && up_tiles * parts * ((width + 4 * pl.ncols - 1) / (4 * pl.ncols)) < 2 * cus;) pl.ncols /= 2;
    pl.nchunk = (width + 4 * pl.ncols - 1) / (4 * pl.ncols);
    pl.up_slots = upto(2 * cus / (up_tiles * parts * pl.nchunk), 1, distinct(16 * LR_MT));
    return pl;
}

// One launch (k_lr_small) for at most 16 rows whose adapter and own rows are few
// values: every workgroup reads them (16 adapters of rank 16, a row each, K and N 4096:
// 9.6 us).  The GPU's time decides, as in a replayed graph or behind other work: one
// against two launches, us per call (N 4096; where the host is what is waited for, the second
// launch costs 2.4 more): R 8, 8 rows each, K 1024 (16384 values) 4.6 / 6.8; R 16, 1 row, K 4096
// (69632) 9.1 / 9.3; 4 rows each (81920) 8.8 / 7.8; R 16, 1 row, K 12288 (208896) 17.9 / 10.9.
constexpr int64_t LR_SMALL = 72 * 1024;
static bool lr_small(int64_t M, int64_t seq, int64_t K, int64_t R) {
    return M <= 16 && R <= 64 && (R + (seq < M ? seq : M)) * K <= LR_SMALL;
}

// The K chunks of a problem do not depend on N or the adapters.
static int64_t lr_chunks(int64_t M, int64_t K, int64_t PR) { return lr_plan(M, 1, K, PR, 8, 1, 1).chunks; }

// Whether rows of out share memory with the rows of t, (M, W): ranges that meet, other than
// other columns of one buffer.
static bool lr_shares(const void *out, int64_t ldo, int64_t N, const void *t, int64_t ldt, int64_t W, int64_t M) {
    const int64_t d = (int64_t)((intptr_t)t - (intptr_t)out) / 2;  // both 16-byte aligned
    if (d >= (M - 1) * ldo + N || -d >= (M - 1) * ldt + W) return false;
    if (M == 1 || ldt != ldo) return true;
    const int64_t col = (d % ldo + ldo) % ldo;
    return col < N || col + W > ldo;
}

}  // namespace qim

using namespace qim;

extern "C" int64_t qim_low_rank_workspace_bytes(int64_t M, int64_t seq, int64_t K, int64_t R, int64_t parts) {
    if (M <= 0 || seq <= 0 || K <= 0 || R <= 0 || parts <= 0 || M >= (1ll << 31) || K >= (1ll << 24) || parts >= (1ll << 14) ||
        R >= (1ll << 14) || parts * R >= (1ll << 14) || lr_small(M, seq, K, R))
        return 0;
    return lr_chunks(M, K, parts * R) * M * parts * R * 4;
}

extern "C" int qim_low_rank(const void *x, int64_t ldx, const void *down, const void *up, const int32_t *index,
                            const float *scale, const void *base, int64_t ldb, void *out, int64_t ldo, void *workspace,
                            int64_t workspace_bytes, int64_t M, int64_t seq, int64_t K, int64_t N, int64_t R,
                            int64_t parts, int64_t A, void *stream) {
    const char *who = "qim_low_rank";
    QIM_REQUIRE(x && down && up && index && out, QIM_ERR_ARG, "%s: null pointer", who);
    QIM_REQUIRE(M > 0 && seq > 0 && K > 0 && N > 0 && R > 0 && parts > 0 && A > 0, QIM_ERR_SHAPE, "%s: empty problem", who);
    QIM_REQUIRE(K % 8 == 0 && R % 8 == 0 && R <= 128 && N % parts == 0 && (N / parts) % 8 == 0, QIM_ERR_SHAPE,
                "%s: K %lld, rank %lld (at most 128) and N %lld / %lld must be multiples of 8", who, (long long)K,
                (long long)R, (long long)N, (long long)parts);
    QIM_REQUIRE(M < (1ll << 31) && K < (1ll << 24) && N < (1ll << 24) && A < (1ll << 24) && parts * R < (1ll << 14),
                QIM_ERR_SHAPE, "%s: too large", who);
    QIM_REQUIRE(ldx >= K && ldo >= N && (!base || ldb >= N) && ldx % 8 == 0 && ldo % 8 == 0 && (!base || ldb % 8 == 0) &&
                    aligned16(x) && aligned16(down) && aligned16(up) && aligned16(base) && aligned16(out) &&
                    aligned16(workspace) && ((reinterpret_cast<uintptr_t>(index) | reinterpret_cast<uintptr_t>(scale)) & 3u) == 0,
                QIM_ERR_LAYOUT, "%s: rows must be 16-byte aligned", who);
    const int64_t PR = parts * R, width = N / parts;
    const LrPlan pl = lr_plan(M, seq, K, PR, width, parts, A);
    const int64_t need = qim_low_rank_workspace_bytes(M, seq, K, R, parts);
    QIM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), QIM_ERR_ARG,
                "%s: workspace of %lld bytes, this problem needs %lld", who, (long long)workspace_bytes, (long long)need);
    const int64_t up_tiles = (M + 16 * LR_MT - 1) / (16 * LR_MT);
    QIM_REQUIRE(up_tiles * pl.nchunk * parts < (1ll << 32) / 256 && pl.tiles * pl.chunks < (1ll << 32) / (64 * LR_WAVES) &&
                    pl.slots * pl.rblocks < 65536,
                QIM_ERR_SHAPE, "%s: too large", who);
    QIM_REQUIRE(!lr_shares(out, ldo, N, x, ldx, K, M) &&
                    (!base || (base == out && (ldb == ldo || M == 1)) || !lr_shares(out, ldo, N, base, ldb, N, M)),
                QIM_ERR_ARG, "%s: out overlaps x, or base other than as the same rows", who);
    LowRankArgs a{(const uint16_t *)x, (const uint16_t *)down, (const uint16_t *)up, (const uint16_t *)base, index, scale,
                  (uint16_t *)out, (float *)workspace, ldx, ldb, ldo, M, (uint32_t)(seq < M ? seq : M), (int)K, (int)N, (int)R,
                  (int)PR, (int)parts, (int)A, (int)pl.chunks, (int)pl.kchunk, pl.ncols, (int)pl.nchunk};
    if (lr_small(M, seq, K, R)) {
        a.nchunk = (int)((width + 511) / 512);
        const int64_t slots = seq > 1 ? (M + seq - 1) / seq : M;
        launch(R <= 16 ? k_lr_small<1, true> : R <= 32 ? k_lr_small<1, false> : k_lr_small<2, false>,
               dim3((unsigned)(a.nchunk * parts), (unsigned)(slots < A ? slots : A)), dim3(512), 0, as_stream(stream), a);
        return check_launch(who);
    }
    using Down = void (*)(LowRankArgs, int);
    static const Down downs[4][3] = {{k_lr_down<1, 1>, k_lr_down<1, 2>, k_lr_down<1, 4>},
                                     {k_lr_down<2, 1>, k_lr_down<2, 2>, k_lr_down<2, 4>},
                                     {k_lr_down<4, 1>, nullptr, k_lr_down<4, 4>},
                                     {k_lr_down<8, 1>, k_lr_down<8, 2>, nullptr}};
    static std::atomic<bool> configured[4][3][QIM_MAX_DEVICES] = {};
    const int ri = pl.rt == 8 ? 3 : pl.rt / 2, mi = pl.mt / 2, lds = LR_WAVES * pl.mt * pl.rt * 64 * 16;
    const Down dn = downs[ri][mi];
    if (lds > 65536)
        if (const int rc = reserve_lds(reinterpret_cast<const void *>(dn), lds, configured[ri][mi], who)) return rc;
    launch(dn, dim3((unsigned)(pl.tiles * pl.chunks), (unsigned)(pl.slots * pl.rblocks)), dim3(64 * LR_WAVES), lds, as_stream(stream), a,
           (int)pl.rblocks);
    void (*const up_fn)(LowRankArgs) = R <= 16 ? k_lr_up<1, true> : R <= 32 ? k_lr_up<1, false> : R <= 64 ? k_lr_up<2, false> : k_lr_up<4, false>;
    launch(up_fn, dim3((unsigned)(up_tiles * pl.nchunk * parts), (unsigned)pl.up_slots), dim3(256), 0,
           as_stream(stream), a);
    return check_launch(who);
}
