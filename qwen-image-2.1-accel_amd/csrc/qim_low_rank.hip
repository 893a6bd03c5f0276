// Low-rank adapters of several requests beside one shared projection:
//
//   out[m] = base[m] + scale[a] * up[a] (down[a] x[m]),   a = index[m / seq]
//
// in two launches.  k_lr_down: h = down x, (M, parts * R) in fp32, with the K
// axis cut into chunks where there are few rows (each chunk's sums go to the
// workspace).  k_lr_up: adds the chunks, multiplies by up and adds to base.
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
// and are bound by that.
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
    int64_t ldx, ldb, ldo, M, seq;
    int K, N, R, PR, parts, A;
    int chunks, kchunk;  // K chunks of kchunk values
    int ncols;           // columns of a block of `out` per workgroup (k_lr_up)
    int nchunk;          // workgroups per part
};

// The adapter of row m, -1 for none.
__device__ __forceinline__ int lr_adapter(const LowRankArgs &p, int64_t m) {
    if (m >= p.M) return -1;
    const int a = p.index[p.seq == 1 ? m : m / p.seq];
    return a >= 0 && a < p.A ? a : -1;
}

// Calls f(a) for each distinct adapter a >= 0 among the lanes' values.
template <class F>
__device__ __forceinline__ void lr_each(int mine, F &&f) {
    uint64_t todo = __builtin_amdgcn_ballot_w64(mine >= 0);
    while (todo) {
        const int a = __builtin_amdgcn_readlane(mine, (int)__builtin_ctzll(todo));
        f(a);
        todo &= ~__builtin_amdgcn_ballot_w64(mine == a);
    }
}

// h of one 16-row tile, one K chunk and 16 * RT rows of down: the 4 waves take
// 32-value steps of the chunk in turn and join in LDS.
template <int RT>
__global__ __launch_bounds__(256) void k_lr_down(LowRankArgs p) {
    __shared__ f32x4_t sum[4][RT][64];
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t m = (int64_t)blockIdx.x * 16 + lr;
    const int r0 = blockIdx.z * (16 * RT);
    const int mine = lr_adapter(p, m);
    const int64_t mc = m < p.M ? m : p.M - 1;
    const int k0 = blockIdx.y * p.kchunk, k1 = k0 + p.kchunk < p.K ? k0 + p.kchunk : p.K;
    const uint16_t *xr = p.x + mc * p.ldx;
    f32x4_t keep[RT] = {};
    lr_each(mine, [&](int a) {
        f32x4_t acc[RT] = {};
        const uint16_t *dn = p.down + (int64_t)a * p.PR * p.K;
        for (int k = k0 + 32 * wave + 8 * kg; k - 8 * kg < k1; k += 128) {
            const bool in = k < k1;
            const u32x4_t zero = {0, 0, 0, 0};
            const u32x4_t xv = in ? *reinterpret_cast<const u32x4_t *>(xr + k) : zero;
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                int r = r0 + 16 * t + lr;
                r = r < p.PR ? r : p.PR - 1;
                const u32x4_t dv = in ? *reinterpret_cast<const u32x4_t *>(dn + (int64_t)r * p.K + k) : zero;
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, dv), __builtin_bit_cast(bf16x8_t, xv),
                                                                 acc[t], 0, 0, 0);
            }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) keep[t][i] = mine == a ? acc[t][i] : keep[t][i];
    });
#pragma unroll
    for (int t = 0; t < RT; ++t) sum[wave][t][lane] = keep[t];
    __syncthreads();
    for (int i = tid; i < RT * 64; i += 256) {
        const int t = i >> 6, l = i & 63;
        const f32x4_t s = (sum[0][t][l] + sum[1][t][l]) + (sum[2][t][l] + sum[3][t][l]);
        // Lane l of the tile: row l % 16, values 4 (l / 16) .. + 3 of its 16.
        const int64_t row = (int64_t)blockIdx.x * 16 + (l & 15);
        const int r = r0 + 16 * t + 4 * (l >> 4);
        if (row < p.M && r < p.PR)
            *reinterpret_cast<f32x4_t *>(p.h + ((int64_t)blockIdx.y * p.M + row) * p.PR + r) = s;
    }
}

// Columns [c0, c0 + ncols) of one part, 16 rows per wave (the workgroup's 4
// waves take neighbouring rows).  STEPS * 32 operand slots: chunks of 8 of hi, then of
// lo.  Two MFMA tiles at a time, whose rows are assigned to columns so that a
// lane's 8 results are 8 neighbouring columns: row i of tile t is column
// 8 (i / 4) + 4 t + i % 4.
template <int STEPS>
__global__ __launch_bounds__(256) void k_lr_up(LowRankArgs p) {
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t m = ((int64_t)blockIdx.x * 4 + wave) * 16 + lr;
    const int part = blockIdx.y / p.nchunk, width = p.N / p.parts;
    const int c0 = (blockIdx.y - part * p.nchunk) * p.ncols, c1 = c0 + p.ncols < width ? c0 + p.ncols : width;
    const int mine = lr_adapter(p, m);
    const float sc = mine >= 0 ? (p.scale ? p.scale[mine] : 1.0f) : 0.0f;
    const int rc = p.R / 8;  // chunks of 8
    bf16x8_t hop[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int ch = 4 * s + kg;
        float f[8] = {};
        if (ch < 2 * rc && mine >= 0) {
            const float *src = p.h + m * p.PR + part * p.R + (ch < rc ? ch : ch - rc) * 8;
            for (int c = 0; c < p.chunks; ++c) {
                const f32x4_t a = *reinterpret_cast<const f32x4_t *>(src), b = *reinterpret_cast<const f32x4_t *>(src + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f[e] += a[e];
                    f[4 + e] += b[e];
                }
                src += p.M * p.PR;
            }
        }
        if (ch >= rc) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float hi = rbf(f[e]);
                f[e] = __builtin_isfinite(hi) ? f[e] - hi : 0.0f;
            }
        }
        hop[s] = __builtin_bit_cast(bf16x8_t, pack8(f));
    }
    for (int c = c0; c < c1; c += 32) {
        f32x4_t keep[2] = {};
        lr_each(mine, [&](int a) {
            f32x4_t acc[2] = {};
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                int n = c + 8 * (lr >> 2) + 4 * t + (lr & 3);
                n = n < width ? n : width - 1;
                const uint16_t *up = p.up + ((int64_t)a * p.N + part * width + n) * p.R;
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    const int ch = 4 * s + kg;
                    const u32x4_t zero = {0, 0, 0, 0};
                    const u32x4_t u = ch < 2 * rc ? *reinterpret_cast<const u32x4_t *>(up + (ch < rc ? ch : ch - rc) * 8) : zero;
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, u), hop[s], acc[t], 0, 0, 0);
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) keep[t][i] = mine == a ? acc[t][i] : keep[t][i];
        });
        const int col = c + 8 * kg;
        if (m < p.M && col < c1) {
            const int64_t n = (int64_t)part * width + col;
            float y[8] = {};
            if (p.base) unpack8(*reinterpret_cast<const uint4 *>(p.base + m * p.ldb + n), y);
            if (mine >= 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[e] = __builtin_fmaf(sc, keep[0][e], y[e]);
                    y[4 + e] = __builtin_fmaf(sc, keep[1][e], y[4 + e]);
                }
            }
            *reinterpret_cast<uint4 *>(p.out + m * p.ldo + n) = pack8(y);
        }
    }
}

// K chunks: as many as bring the first launch to two workgroups per CU, each
// with at least 128 values (one step per wave).
static int64_t lr_chunks(int64_t M, int64_t K, int64_t PR) {
    const int64_t cus = device_cus() > 0 ? device_cus() : 256;
    const int64_t tiles = (M + 15) / 16 * ((PR + 127) / 128);
    int64_t n = 2 * cus / tiles;
    const int64_t most = (K + 127) / 128;
    n = n < most ? n : most;
    n = n < 16 ? n : 16;
    return n > 1 ? n : 1;
}

}  // namespace qim

using namespace qim;

extern "C" int64_t qim_low_rank_workspace_bytes(int64_t M, int64_t K, int64_t R) {
    if (M <= 0 || K <= 0 || R <= 0 || M >= (1ll << 31) || K >= (1ll << 24) || R >= (1ll << 14)) return 0;
    return lr_chunks(M, K, R) * M * R * 4;
}

extern "C" int qim_low_rank(const void *x, int64_t ldx, const void *down, const void *up, const int32_t *index,
                            const float *scale, const void *base, int64_t ldb, void *out, int64_t ldo, void *workspace,
                            int64_t workspace_bytes, int64_t M, int64_t seq, int64_t K, int64_t N, int64_t R,
                            int64_t parts, int64_t A, void *stream) {
    const char *who = "qim_low_rank";
    QIM_REQUIRE(x && down && up && index && out && workspace, QIM_ERR_ARG, "%s: null pointer", who);
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
    const int64_t PR = parts * R, chunks = lr_chunks(M, K, PR);
    QIM_REQUIRE(workspace_bytes >= chunks * M * PR * 4, QIM_ERR_ARG, "%s: workspace of %lld bytes, this problem needs %lld", who,
                (long long)workspace_bytes, (long long)(chunks * M * PR * 4));
    LowRankArgs a{(const uint16_t *)x, (const uint16_t *)down, (const uint16_t *)up, (const uint16_t *)base, index, scale,
                  (uint16_t *)out, (float *)workspace, ldx, ldb, ldo, M, seq, (int)K, (int)N, (int)R, (int)PR, (int)parts,
                  (int)A, (int)chunks, (int)(((K + chunks - 1) / chunks + 127) / 128 * 128), 0, 0};
    a.chunks = (int)((K + a.kchunk - 1) / a.kchunk);  // none empty after rounding
    const int64_t width = N / parts;
    a.ncols = 256;
    a.nchunk = (int)((width + a.ncols - 1) / a.ncols);
    QIM_REQUIRE((int64_t)a.nchunk * parts < 65536, QIM_ERR_SHAPE, "%s: too many columns", who);
    const int64_t rt = PR <= 16 ? 1 : PR <= 32 ? 2 : PR <= 64 ? 4 : 8;
    void (*const dn)(LowRankArgs) = rt == 1 ? k_lr_down<1> : rt == 2 ? k_lr_down<2> : rt == 4 ? k_lr_down<4> : k_lr_down<8>;
    launch(dn, dim3((unsigned)((M + 15) / 16), (unsigned)a.chunks, (unsigned)((PR + 16 * rt - 1) / (16 * rt))), dim3(256), 0, as_stream(stream), a);
    const int steps = R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8;
    void (*const up_fn)(LowRankArgs) = steps == 1 ? k_lr_up<1> : steps == 2 ? k_lr_up<2> : steps == 4 ? k_lr_up<4> : k_lr_up<8>;
    launch(up_fn, dim3((unsigned)((M + 63) / 64), (unsigned)(a.nchunk * parts)), dim3(256), 0, as_stream(stream), a);
    return check_launch(who);
}
