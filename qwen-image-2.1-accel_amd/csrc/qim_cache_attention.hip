// Attention of a few tokens over a K/V cache in MXFP8 (qim_cache.hip): one
// token of each request, or up to 64 drafted ones with a tree mask, head dim
// 128, query heads in groups of G that share a K/V head.
//
//   o[r] = sum_t p_rt V[t] / sum_t p_rt,  p_rt = 2^(c q_r . K[t] - m_r)
//
// in one pass over the keys with a running maximum m_r and sum (fp32).  The
// S * G query rows that share a K/V head are the columns of the MFMA tiles, so
// a key is read once for up to 64 of them.  A row costs 512 flop for a
// key's 264 bytes; up to about a hundred rows the cache's bytes bound it.
//
// Transposed products on v_mfma_f32_32x32x16_bf16, 32 keys at a time: S^T = K Q^T
// (32 keys x 32 rows) and O^T = V^T P^T (32 head dims x 32 rows), so a lane owns
// query row lane % 32 in both, m and the sum are lane-local, and the S^T
// accumulator is already the B operand of the second product (lane (row, hf)
// holds keys 8(i/4) + 4hf + i%4, i = 0..15).  Codes become bf16 exactly (4
// significand bits times a power of two), with the block's exponent as the
// conversion's scale operand.  K goes from memory to the A operand as it is:
// lane (key, hf) loads the 16 codes [32j + 16hf, +16) for each j, whose two
// halves are two 8-value operands; Q is held in the same order (an MFMA pairs
// the K slots of A and B by position).  V is converted into a per-wave LDS tile
// of 32 keys x 128 and transposed by the LDS reads.
//
// Work split: a workgroup is one (sequence, K/V head, row tile, key chunk); its
// 4 waves take 32-key blocks of the chunk in turn, each with its own running
// maximum, and join in LDS.  Where there are too few (sequence, head) pairs to
// fill the chip the keys are cut into nsplit chunks (of the sequence's
// own length, read on the device) and a second launch joins them.
#include "qim_device.h"
#include "qim_runtime.h"

namespace qim {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16a_t __attribute__((ext_vector_type(16)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

constexpr int CA_D = 128;
constexpr int CA_KB = 32;                        // keys per block
constexpr int CA_VTILE = CA_KB * CA_D * 2;       // 8 KiB of LDS per wave
constexpr int CA_OROW = CA_D + 4;                // floats per row of the joining buffer (staggers the banks)
constexpr int CA_MAX_S = 64;
constexpr int CA_MAX_SPLIT = 64;

struct CacheAttnArgs {
    const uint16_t *q;
    int64_t ldqb, ldq;
    const uint8_t *kc, *ks, *vc, *vs;
    const int32_t *lengths;
    const uint8_t *tree;
    int64_t tree_b;
    uint16_t *o;
    float *part_o;   // (item, split, row of the tile, 128), relative to the split's maximum
    float2 *part_ml; // (item, split, row of the tile): (maximum, sum)
    int64_t C;
    int S, H, HK, G, rows, ntile, nsplit;
    float scale_log2e;
};

// The bf16 operand of 8 codes of a block.
__device__ __forceinline__ bf16x8_t ca_operand(uint32_t lo, uint32_t hi, float scale) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 32 keys of K and V as loaded: K of lane (key = lane % 32, hf) chunks 2j + hf;
// V of lane: key 8 it + lane / 8, chunk lane % 8.
struct CaRaw {
    uint4 k[4], v[4];
    uint32_t ks, vs[4];
};

__device__ __forceinline__ float ca_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float ca_swap_max(float x) {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return ca_max(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

template <int NT>
__global__ __launch_bounds__(256) void k_cache_attn(CacheAttnArgs p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Neighbouring workgroups: the row tiles of a head (which share its keys in
    // L2), then the heads (whose 128-byte pieces are neighbours in memory).
    const int item = blockIdx.x, split = blockIdx.y;
    const int tile = item % p.ntile, h = (item / p.ntile) % p.HK, b = item / (p.ntile * p.HK);
    const int64_t len64 = p.lengths[b];
    const int64_t len = len64 < 0 ? 0 : len64 > p.C ? p.C : len64;
    const int64_t nblk = (len + CA_KB - 1) / CA_KB, per = (nblk + p.nsplit - 1) / p.nsplit;
    const int64_t blk0 = split * per, blk1 = blk0 + per < nblk ? blk0 + per : nblk;
    const int row0 = tile * 32 * NT;
    const float c = p.scale_log2e;
    const float ninf = -__builtin_inff();

    // Q operands, and the tree's bits of each row.
    bf16x8_t qf[NT][8];
    uint64_t bits[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        int r = row0 + 32 * t + lq;
        r = r < p.rows ? r : p.rows - 1;  // rows past the end: computed, not stored
        const int s = r / p.G, head = h * p.G + (r - s * p.G);
        const uint16_t *qr = p.q + b * p.ldqb + s * p.ldq + head * CA_D + hf * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            qf[t][2 * j] = *reinterpret_cast<const bf16x8_t *>(qr + 32 * j);
            qf[t][2 * j + 1] = *reinterpret_cast<const bf16x8_t *>(qr + 32 * j + 8);
        }
        bits[t] = 0;
        if (p.tree) {
            const uint8_t *mask = p.tree + b * p.tree_b + s * p.S;
            for (int j = 0; j < p.S; ++j) bits[t] |= (uint64_t)(mask[j] != 0) << j;
        }
    }

    f32x16a_t o[NT][4];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = ninf;
        l[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) o[t][dt] = f32x16a_t{};
    }

    const int64_t W = (int64_t)p.HK * CA_D;
    const uint8_t *kc = p.kc + b * p.C * W + h * CA_D, *vc = p.vc + b * p.C * W + h * CA_D;
    const uint8_t *ks = p.ks + (b * p.C * W + h * CA_D) / 32, *vs = p.vs + (b * p.C * W + h * CA_D) / 32;
    auto load = [&](int64_t blk, CaRaw &x) {
        const int64_t k0 = blk * CA_KB;
        int64_t key = k0 + lq;
        key = key < p.C ? key : p.C - 1;
        const uint8_t *at = kc + key * W + hf * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) x.k[j] = *reinterpret_cast<const uint4 *>(at + 32 * j);
        x.ks = *reinterpret_cast<const uint32_t *>(ks + key * (W / 32));
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            int64_t vk = k0 + 8 * it + (lane >> 3);
            vk = vk < p.C ? vk : p.C - 1;
            x.v[it] = *reinterpret_cast<const uint4 *>(vc + vk * W + (lane & 7) * 16);
            x.vs[it] = *reinterpret_cast<const uint32_t *>(vs + vk * (W / 32));
        }
    };

    // This wave's V tile.  Row = key, 16-byte chunk c at chunk c ^ 4 (key % 4).
    uint8_t *const vt = lds + wave * CA_VTILE;
    const uint32_t vbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)vt;
    uint32_t vread[4];
    {
        const int i = lane & 15;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
            vread[dt] = vbase + (4 * hf + (i >> 2)) * 256 + ((dt ^ (i >> 2)) << 6) + ((lane >> 4) & 1) * 32 + (i & 3) * 8;
    }

    const int64_t tree0 = p.tree ? len - p.S : len;  // the first key that needs a look at the mask
    CaRaw cur, nxt;
    if (blk0 + wave < blk1) load(blk0 + wave, cur);
    for (int64_t blk = blk0 + wave; blk < blk1; blk += 4) {
        const int64_t k0 = blk * CA_KB;
        if (blk + 4 < blk1) load(blk + 4, nxt);
        // V rows past the last key are zeros, whatever the cache holds there.
        const int shift = 8 * ((lane & 7) >> 1);
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const int key = 8 * it + (lane >> 3), ch = 2 * (lane & 7);
            const bool in = k0 + key < len;
            const float s = mx_scale_operand(in ? (int)((cur.vs[it] >> shift) & 0xffu) : 0);
            const uint4 x = in ? cur.v[it] : make_uint4(0, 0, 0, 0);
            uint8_t *row = vt + key * 256;
            *reinterpret_cast<bf16x8_t *>(row + ((ch ^ ((key & 3) << 2)) << 4)) = ca_operand(x.x, x.y, s);
            *reinterpret_cast<bf16x8_t *>(row + (((ch + 1) ^ ((key & 3) << 2)) << 4)) = ca_operand(x.z, x.w, s);
        }
        f32x16a_t s[NT];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float sc = mx_scale_operand((int)((cur.ks >> (8 * j)) & 0xffu));
            const bf16x8_t a = ca_operand(cur.k[j].x, cur.k[j].y, sc), bq = ca_operand(cur.k[j].z, cur.k[j].w, sc);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qf[t][2 * j], j == 0 ? f32x16a_t{} : s[t], 0, 0, 0);
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bq, qf[t][2 * j + 1], s[t], 0, 0, 0);
            }
        }
        // Only blocks that reach the tree's keys or the end have anything masked.
        const bool masked = k0 + CA_KB > tree0;
        uint32_t seen[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            seen[t] = ~0u;
            if (masked) {
                // The block's 32 keys as bits: keys before the tree's are seen.
                const int64_t s0 = k0 - tree0, left = len - k0;  // s0 > -32, left >= 1
                uint32_t w = s0 >= 0 ? (uint32_t)(bits[t] >> s0)
                                     : ((uint32_t)bits[t] << (uint32_t)-s0) | ((1u << (uint32_t)-s0) - 1u);
                if (left < 32) w &= (1u << (uint32_t)left) - 1u;
                seen[t] = w >> (4 * hf);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = (seen[t] >> (8 * (i >> 2) + (i & 3))) & 1u ? s[t][i] : ninf;
            }
        }
        uint32_t pw[NT][8];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float mx = ca_max(s[t][0], s[t][1]);
#pragma unroll
            for (int i = 2; i < 16; ++i) mx = ca_max(mx, s[t][i]);
            mx = ca_swap_max(mx) * c;
            const float mn = ca_max(m[t], mx);
            const float ref = mn == ninf ? 0.f : mn;  // nothing seen yet: every p is 0
            const float alpha = __builtin_amdgcn_exp2f(m[t] - ref);
            m[t] = mn;
            float e[16], sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], c, -ref));
                sum += e[i];
            }
            l[t] = l[t] * alpha + sum;
            // p is rounded to bf16 for the matrix product: at most 2^-9 of each
            // term of a sum that is itself rounded to bf16 at the end.
#pragma unroll
            for (int i = 0; i < 8; ++i) pw[t][i] = pack_bf16x2(e[2 * i], e[2 * i + 1]);
            if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) o[t][dt] *= alpha;
            }
        }
        // A wave's LDS operations run in order; the compiler must not reorder them.
        asm volatile("" ::: "memory");
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
            typedef __attribute__((address_space(3))) i16x4_t *ptr_t;
            bf16x8_t vf[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t at = vread[dt] + u * (16 * CA_D * 2);
                const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<ptr_t>((uintptr_t)at));
                const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<ptr_t>((uintptr_t)(at + 8 * CA_D * 2)));
                vf[u] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            }
            if (masked) {
                // A key that one row does not see may hold infinities or NaN for
                // another: those values leave the product (0 * NaN is NaN) and make
                // NaN of the rows that do see their key, by a product of
                // "not finite" and "seen".
                typedef unsigned int u4 __attribute__((ext_vector_type(4)));
                u4 ind[2];
                bool any = false;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    u4 w = __builtin_bit_cast(u4, vf[u]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t lo = (w[e] & 0x7f80u) == 0x7f80u ? 0x3f80u : 0u;
                        const uint32_t hi = (w[e] & 0x7f800000u) == 0x7f800000u ? 0x3f800000u : 0u;
                        ind[u][e] = lo | hi;
                        if (lo) w[e] &= 0xffff0000u;
                        if (hi) w[e] &= 0x0000ffffu;
                        any |= ind[u][e] != 0;
                    }
                    vf[u] = __builtin_bit_cast(bf16x8_t, w);
                }
                if (__builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        f32x16a_t hit{};
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            u4 sv;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t two = seen[t] >> (16 * u + 8 * (e >> 1) + 2 * (e & 1));
                                sv[e] = ((two & 1u) ? 0x3f80u : 0u) | ((two & 2u) ? 0x3f800000u : 0u);
                            }
                            hit = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, ind[u]),
                                                                         __builtin_bit_cast(bf16x8_t, sv), hit, 0, 0, 0);
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            o[t][dt][i] = hit[i] > 0.f ? __builtin_nanf("") : o[t][dt][i];
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const u32x4_t w = {pw[t][4 * u], pw[t][4 * u + 1], pw[t][4 * u + 2], pw[t][4 * u + 3]};
                    o[t][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[u], __builtin_bit_cast(bf16x8_t, w), o[t][dt], 0, 0, 0);
                }
        }
        asm volatile("" ::: "memory");
        cur = nxt;
    }

    // Join the four waves: weights 2^(m_w - M), then the sums, a tile at a time.
    float *const buf = reinterpret_cast<float *>(lds);                        // [4][32][CA_OROW]
    float2 *const ml = reinterpret_cast<float2 *>(buf + 4 * 32 * CA_OROW);    // [4][32]
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        __syncthreads();  // the V tiles, or the previous tile, are done with
        const float lt = l[t] + __shfl_xor(l[t], 32, 64);
        if (hf == 0) ml[wave * 32 + lq] = make_float2(m[t], lt);
        __syncthreads();
        float M = ca_max(ca_max(ml[lq].x, ml[32 + lq].x), ca_max(ml[64 + lq].x, ml[96 + lq].x));
        M = M == ninf ? 0.f : M;
        const float wgt = __builtin_amdgcn_exp2f(m[t] - M);
        float *row = buf + (wave * 32 + lq) * CA_OROW;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4 *>(row + 32 * dt + 8 * g + 4 * hf) =
                    make_float4(o[t][dt][4 * g] * wgt, o[t][dt][4 * g + 1] * wgt, o[t][dt][4 * g + 2] * wgt, o[t][dt][4 * g + 3] * wgt);
        __syncthreads();
        // 8 threads per row, 16 head dims each.
        const int rl = tid >> 3, d0 = (tid & 7) * 16, r = row0 + 32 * t + rl;
        float acc[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] = 0.f;
        float Mr = ninf, L = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) Mr = ca_max(Mr, ml[w * 32 + rl].x);
        const float Mz = Mr == ninf ? 0.f : Mr;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 x = ml[w * 32 + rl];
            L += x.y * __builtin_amdgcn_exp2f(x.x - Mz);
            const float *src = buf + (w * 32 + rl) * CA_OROW + d0;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(src + e);
                acc[e] += f.x;
                acc[e + 1] += f.y;
                acc[e + 2] += f.z;
                acc[e + 3] += f.w;
            }
        }
        if (r < p.rows) {
            if (p.nsplit == 1) {
                const float inv = L == 0.f ? 0.f : 1.0f / L;  // no visible key: zeros
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[e] *= inv;
                const int s = r / p.G, head = h * p.G + (r - s * p.G);
                uint16_t *dst = p.o + (((int64_t)b * p.S + s) * p.H + head) * CA_D + d0;
                *reinterpret_cast<uint4 *>(dst) = pack8(acc);
                *reinterpret_cast<uint4 *>(dst + 8) = pack8(acc + 8);
            } else {
                const int64_t at = ((int64_t)item * p.nsplit + split) * (32 * NT) + 32 * t + rl;
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4 *>(p.part_o + at * CA_D + d0 + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
                if ((tid & 7) == 0) p.part_ml[at] = make_float2(Mr, L);
            }
        }
    }
}

// Join the key chunks: 32 lanes per row, 4 head dims each.
__global__ __launch_bounds__(256) void k_cache_attn_join(CacheAttnArgs p, int tile_rows, int64_t nrows) {
    const int64_t g = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int d0 = (threadIdx.x & 31) * 4;
    if (g >= nrows) return;
    const int64_t item0 = g / p.rows;  // (sequence, K/V head)
    const int r = (int)(g - item0 * p.rows), tile = r / tile_rows, rl = r - tile * tile_rows;
    const int64_t first = ((item0 * p.ntile + tile) * p.nsplit) * tile_rows + rl;
    float M = -__builtin_inff();
    for (int i = 0; i < p.nsplit; ++i) M = ca_max(M, p.part_ml[first + (int64_t)i * tile_rows].x);
    M = M == -__builtin_inff() ? 0.f : M;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float L = 0.f;
    for (int i = 0; i < p.nsplit; ++i) {
        const int64_t at = first + (int64_t)i * tile_rows;
        const float2 ml = p.part_ml[at];
        const float4 f = *reinterpret_cast<const float4 *>(p.part_o + at * CA_D + d0);
        const float w = __builtin_amdgcn_exp2f(ml.x - M);
        L += ml.y * w;
        acc.x += f.x * w;
        acc.y += f.y * w;
        acc.z += f.z * w;
        acc.w += f.w * w;
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    const int h = (int)(item0 % p.HK), s = r / p.G, head = h * p.G + (r - s * p.G);
    uint16_t *dst = p.o + (((item0 / p.HK) * p.S + s) * p.H + head) * CA_D + d0;
    *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

// Row tiles of 32 (one MFMA tile) or 64, and key chunks: as many as bring the
// launch to two workgroups per CU, each with at least a block for every wave.
struct CaPlan {
    int64_t rows, tile, ntile, items, nsplit;
    int64_t part_o() const { return nsplit > 1 ? items * nsplit * tile * CA_D * 4 : 0; }
    int64_t bytes() const { return nsplit > 1 ? part_o() + items * nsplit * tile * 8 : 0; }
};
static CaPlan ca_plan(int64_t B, int64_t S, int64_t C, int64_t H, int64_t HK) {
    CaPlan pl;
    pl.rows = S * (H / HK);
    pl.tile = pl.rows > 32 ? 64 : 32;
    pl.ntile = (pl.rows + pl.tile - 1) / pl.tile;
    pl.items = B * HK * pl.ntile;
    const int64_t cus = device_cus() > 0 ? device_cus() : 256, nblk = (C + CA_KB - 1) / CA_KB;
    int64_t n = (2 * cus + pl.items - 1) / pl.items;
    const int64_t most = nblk / 4;
    n = n < most ? n : most;
    n = n < CA_MAX_SPLIT ? n : CA_MAX_SPLIT;
    pl.nsplit = n > 1 ? n : 1;
    return pl;
}

}  // namespace qim

using namespace qim;

static bool ca_shape(int64_t B, int64_t S, int64_t C, int64_t H, int64_t HK) {
    return B > 0 && S > 0 && S <= CA_MAX_S && C > 0 && C < (1ll << 31) && HK > 0 && H > 0 && H % HK == 0 && H <= (1 << 16) && B < (1 << 20) &&
           B * HK * ((S * (H / HK) + 31) / 32) < (1 << 24);
}

extern "C" int64_t qim_attention_cached_workspace_bytes(int64_t B, int64_t S, int64_t C, int64_t H, int64_t HK) {
    return ca_shape(B, S, C, H, HK) ? ca_plan(B, S, C, H, HK).bytes() : 0;
}

extern "C" int qim_attention_cached(const void *q, int64_t ldqb, int64_t ldq, const void *kc, const void *ks,
                                    const void *vc, const void *vs, const int32_t *lengths, const void *tree,
                                    int64_t tree_b, void *o, void *workspace, int64_t workspace_bytes, int64_t B,
                                    int64_t S, int64_t C, int64_t H, int64_t HK, int64_t D, float scale, void *stream) {
    const char *who = "qim_attention_cached";
    QIM_REQUIRE(q && kc && ks && vc && vs && lengths && o, QIM_ERR_ARG, "%s: null pointer", who);
    QIM_REQUIRE(D == CA_D, QIM_ERR_SHAPE, "%s: head dim %lld (128 only)", who, (long long)D);
    QIM_REQUIRE(scale > 0.0f && scale < 1e30f, QIM_ERR_ARG, "%s: scale must be positive and finite", who);
    QIM_REQUIRE(ca_shape(B, S, C, H, HK), QIM_ERR_SHAPE,
                "%s: B %lld, S %lld (1..64), C %lld, %lld heads on %lld K/V heads", who, (long long)B, (long long)S,
                (long long)C, (long long)H, (long long)HK);
    QIM_REQUIRE(ldq >= H * D && ldqb >= 0 && ldq % 8 == 0 && ldqb % 8 == 0 && tree_b >= 0 && aligned16(q) && aligned16(kc) &&
                    aligned16(ks) && aligned16(vc) && aligned16(vs) && aligned16(o) && (reinterpret_cast<uintptr_t>(lengths) & 3u) == 0,
                QIM_ERR_LAYOUT, "%s: rows must be 16-byte aligned", who);
    const CaPlan pl = ca_plan(B, S, C, H, HK);
    QIM_REQUIRE(pl.bytes() == 0 || (workspace && workspace_bytes >= pl.bytes()), QIM_ERR_ARG,
                "%s: workspace of %lld bytes, this problem needs %lld", who, (long long)workspace_bytes, (long long)pl.bytes());
    QIM_REQUIRE(aligned16(workspace), QIM_ERR_LAYOUT, "%s: workspace must be 16-byte aligned", who);
    static std::atomic<bool> configured[2][QIM_MAX_DEVICES] = {};
    constexpr int bytes = (4 * 32 * CA_OROW) * 4 + 4 * 32 * 8;
    void (*const fn)(CacheAttnArgs) = pl.tile == 64 ? k_cache_attn<2> : k_cache_attn<1>;
    if (const int rc = reserve_lds(reinterpret_cast<const void *>(fn), bytes, configured[pl.tile == 64], who)) return rc;
    CacheAttnArgs a{(const uint16_t *)q, ldqb, ldq, (const uint8_t *)kc, (const uint8_t *)ks, (const uint8_t *)vc,
                    (const uint8_t *)vs, lengths, (const uint8_t *)tree, tree_b, (uint16_t *)o, (float *)workspace,
                    (float2 *)((uint8_t *)workspace + pl.part_o()), C, (int)S, (int)H, (int)HK, (int)(H / HK),
                    (int)pl.rows, (int)pl.ntile, (int)pl.nsplit, scale * 1.4426950408889634f};
    launch(fn, dim3((unsigned)pl.items, (unsigned)pl.nsplit), dim3(256), bytes, as_stream(stream), a);
    if (pl.nsplit > 1) {
        const int64_t nrows = B * HK * pl.rows;
        launch(k_cache_attn_join, dim3((unsigned)((nrows + 7) / 8)), dim3(256), 0, as_stream(stream), a, (int)pl.tile, nrows);
    }
    return check_launch(who);
}
