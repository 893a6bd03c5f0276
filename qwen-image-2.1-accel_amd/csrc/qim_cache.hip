// A layer's K/V cache in MXFP8: rows quantized as they are written, and read
// back in bf16.
//
// The cache of B sequences holds C positions each: codes (B, C, H, D) E4M3 and
// exponents (B, C, H, D/32) E8M0 bytes, one per 32 values of a head row, for K
// and for V.  A block's exponent and codes are those of qim_mx_quantize
// (mx_exponent, the scaled conversion); D % 32 == 0, so a token's H * D = W
// values are W / 32 blocks whatever the head dim, and both kernels see a token
// as W values.  Reading back is exact: 4 significand bits times a power of two
// is a bf16 value.
//
// Bound by the bytes, each moved once.  Of 4296 tokens of 32 heads of 128 (107 MB):
// written in 20.0 us (5.3 TB/s), read back in 16.7 (6.4 TB/s, part of the codes still
// in the last-level cache); 16 single tokens 3.9 us.
#include "qim_device.h"
#include "qim_runtime.h"

namespace qim {

struct CacheWriteArgs {
    const uint16_t *src[2];   // K and V rows, (B, S, W)
    int64_t ldb[2], ldt[2];   // elements between batches and between tokens
    uint8_t *codes[2], *exps[2];
    const int32_t *start, *count;  // per sequence; null: `first`, S
    int64_t first, S, C, W;
    uint32_t groups;          // waves per token and tensor
    uint32_t waves;
};

// One wave: 64 * U vectors of 8 values of one token of K or of V; 4 lanes hold a
// block.  Rows past count[b], or whose position lies outside [0, C), are not
// written.
constexpr int CACHE_U = 2;
__global__ __launch_bounds__(256) void k_cache_write(CacheWriteArgs p) {
    const int lane = threadIdx.x & 63;
    const uint32_t w = blockIdx.x * 4u + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w >= p.waves) return;
    const uint32_t item = w / p.groups, group = w - item * p.groups;
    const uint32_t token = item >> 1, which = item & 1;
    const uint32_t b = token / (uint32_t)p.S, s = token - b * (uint32_t)p.S;
    if (p.count && (int64_t)s >= p.count[b]) return;
    const int64_t pos = (p.start ? (int64_t)p.start[b] : p.first) + s;
    if (pos < 0 || pos >= p.C) return;
    const uint16_t *src = (which ? p.src[1] : p.src[0]) + b * (which ? p.ldb[1] : p.ldb[0]) + s * (which ? p.ldt[1] : p.ldt[0]);
    const int64_t row = ((int64_t)b * p.C + pos) * p.W;
    uint8_t *codes = (which ? p.codes[1] : p.codes[0]) + row;
    uint8_t *exps = (which ? p.exps[1] : p.exps[0]) + row / 32;
    const uint32_t v0 = group * (64 * CACHE_U) + lane, nv = (uint32_t)(p.W / 8);
    uint4 x[CACHE_U];
#pragma unroll
    for (int u = 0; u < CACHE_U; ++u)
        x[u] = v0 + 64 * u < nv ? ld_nt(src + (int64_t)(v0 + 64 * u) * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < CACHE_U; ++u) {
        int e;
        const uint2 c = quantize8_bf16(x[u], e);  // a block's 4 lanes are all in or all out of the row
        const uint32_t v = v0 + 64 * u;
        if (v < nv) {
            *reinterpret_cast<uint2 *>(codes + (int64_t)v * 8) = c;
            if ((v & 3) == 0) exps[v >> 2] = (uint8_t)e;
        }
    }
}

struct CacheReadArgs {
    const uint8_t *codes[2], *exps[2];
    uint16_t *out[2];
    int64_t C, W, rows;  // positions [0, rows) of each sequence
    uint32_t groups, waves;
};

// One wave: 64 * U vectors of 8 codes of one token of K or of V.
__global__ __launch_bounds__(256) void k_cache_read(CacheReadArgs p) {
    const int lane = threadIdx.x & 63;
    const uint32_t w = blockIdx.x * 4u + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w >= p.waves) return;
    const uint32_t item = w / p.groups, group = w - item * p.groups;
    const uint32_t token = item >> 1, which = item & 1;
    const uint32_t b = token / (uint32_t)p.rows, s = token - b * (uint32_t)p.rows;
    const int64_t row = ((int64_t)b * p.C + s) * p.W;
    const uint8_t *codes = (which ? p.codes[1] : p.codes[0]) + row;
    const uint8_t *exps = (which ? p.exps[1] : p.exps[0]) + row / 32;
    uint16_t *out = (which ? p.out[1] : p.out[0]) + (int64_t)token * p.W;
    const uint32_t v0 = group * (64 * CACHE_U) + lane, nv = (uint32_t)(p.W / 8);
    uint2 c[CACHE_U];
    int e[CACHE_U];
#pragma unroll
    for (int u = 0; u < CACHE_U; ++u) {
        const uint32_t v = v0 + 64 * u;
        if (v < nv) {
            c[u] = *reinterpret_cast<const uint2 *>(codes + (int64_t)v * 8);
            e[u] = exps[v >> 2];
        }
    }
#pragma unroll
    for (int u = 0; u < CACHE_U; ++u) {
        const uint32_t v = v0 + 64 * u;
        if (v < nv) st_nt(out + (int64_t)v * 8, dequantize8(c[u], e[u]));
    }
}

}  // namespace qim

using namespace qim;

static int cache_common(const char *who, const void *kc, const void *ks, const void *vc, const void *vs, int64_t B,
                        int64_t rows, int64_t C, int64_t H, int64_t D) {
    QIM_REQUIRE(kc && ks && vc && vs, QIM_ERR_ARG, "%s: null pointer", who);
    QIM_REQUIRE(B > 0 && rows > 0 && C > 0 && H > 0 && D > 0, QIM_ERR_SHAPE, "%s: empty problem", who);
    QIM_REQUIRE(D % 32 == 0 && D <= 1024 && H <= (1 << 20), QIM_ERR_SHAPE, "%s: %lld heads of %lld (head dims are multiples of 32)", who,
                (long long)H, (long long)D);
    QIM_REQUIRE(B < (1ll << 31) && rows < (1ll << 31) && C < (1ll << 31), QIM_ERR_SHAPE, "%s: too large", who);
    QIM_REQUIRE(aligned16(kc) && aligned16(vc) && aligned16(ks) && aligned16(vs), QIM_ERR_LAYOUT,
                "%s: codes and exponents must be 16-byte aligned", who);
    return QIM_OK;
}

// Waves of 64 * CACHE_U vectors per token and tensor; 0 if the launch is too large
// (2^32 threads or more).
static int64_t cache_grid(int64_t tokens, int64_t W, uint32_t &groups, uint32_t &waves) {
    const int64_t g = (W / 8 + 64 * CACHE_U - 1) / (64 * CACHE_U);
    if (tokens > ((1ll << 26) - 4) / (2 * g)) return 0;
    groups = (uint32_t)g;
    waves = (uint32_t)(tokens * 2 * g);
    return ((int64_t)waves + 3) / 4;
}

extern "C" int qim_cache_write(const void *k, int64_t ldkb, int64_t ldk, const void *v, int64_t ldvb, int64_t ldv,
                               void *kc, void *ks, void *vc, void *vs, const int32_t *start, int64_t first,
                               const int32_t *count, int64_t B, int64_t S, int64_t C, int64_t H, int64_t D,
                               void *stream) {
    QIM_REQUIRE(k && v, QIM_ERR_ARG, "qim_cache_write: null pointer");
    if (int rc = cache_common("qim_cache_write", kc, ks, vc, vs, B, S, C, H, D)) return rc;
    const int64_t W = H * D;
    QIM_REQUIRE(start || (first >= 0 && first <= C - S), QIM_ERR_ARG,
                "qim_cache_write: %lld rows from position %lld of %lld", (long long)S, (long long)first, (long long)C);
    QIM_REQUIRE(ldk >= W && ldv >= W && ldkb >= 0 && ldvb >= 0 && ldk % 8 == 0 && ldv % 8 == 0 && ldkb % 8 == 0 &&
                    ldvb % 8 == 0 && aligned16(k) && aligned16(v),
                QIM_ERR_LAYOUT, "qim_cache_write: k and v rows must be 16-byte aligned and at least H*D apart");
    CacheWriteArgs a{{(const uint16_t *)k, (const uint16_t *)v}, {ldkb, ldvb}, {ldk, ldv}, {(uint8_t *)kc, (uint8_t *)vc},
                     {(uint8_t *)ks, (uint8_t *)vs}, start, count, first, S, C, W, 0, 0};
    const int64_t blocks = B < (1ll << 31) / S ? cache_grid(B * S, W, a.groups, a.waves) : 0;
    QIM_REQUIRE(blocks, QIM_ERR_SHAPE, "qim_cache_write: too large");
    launch(k_cache_write, dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), a);
    return check_launch("qim_cache_write");
}

extern "C" int qim_cache_read(const void *kc, const void *ks, const void *vc, const void *vs, void *ok, void *ov,
                              int64_t B, int64_t C, int64_t rows, int64_t H, int64_t D, void *stream) {
    QIM_REQUIRE(ok && ov, QIM_ERR_ARG, "qim_cache_read: null pointer");
    if (int rc = cache_common("qim_cache_read", kc, ks, vc, vs, B, rows, C, H, D)) return rc;
    QIM_REQUIRE(rows <= C, QIM_ERR_ARG, "qim_cache_read: %lld rows of a cache of %lld", (long long)rows, (long long)C);
    QIM_REQUIRE(aligned16(ok) && aligned16(ov), QIM_ERR_LAYOUT, "qim_cache_read: outputs must be 16-byte aligned");
    CacheReadArgs a{{(const uint8_t *)kc, (const uint8_t *)vc}, {(const uint8_t *)ks, (const uint8_t *)vs},
                    {(uint16_t *)ok, (uint16_t *)ov}, C, H * D, rows, 0, 0};
    const int64_t blocks = B < (1ll << 31) / rows ? cache_grid(B * rows, H * D, a.groups, a.waves) : 0;
    QIM_REQUIRE(blocks, QIM_ERR_SHAPE, "qim_cache_read: too large");
    launch(k_cache_read, dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), a);
    return check_launch("qim_cache_read");
}
