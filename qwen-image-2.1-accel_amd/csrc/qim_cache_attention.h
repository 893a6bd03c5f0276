// Attention over a K/V cache in MXFP8: what the kernels that read such a cache in place share
// (qim_cache_attention.hip, qim_shared_attention.hip).
#pragma once

#include "qim_device.h"

namespace qim {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

constexpr int CA_D = 128;
constexpr int CA_KB = 32;                        // keys per block
constexpr int CA_VTILE = CA_KB * CA_D * 2;       // 8 KiB of LDS per wave
constexpr int CA_MAX_S = 64;

// The bf16 operand of 8 codes of a block.
__device__ __forceinline__ bf16x8_t ca_operand(uint32_t lo, uint32_t hi, float scale) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float ca_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float ca_swap_max(float x) {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return ca_max(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

// The tree's bits of query s: bit j, whether it sees the j-th of the last S keys.
// Four truth bytes per load (rows of S bytes, any alignment), all loads in flight
// together; the last load ends at the row's end and repeats bits.
// row: the S truth bytes of the query, or NULL (0).
__device__ __forceinline__ uint64_t ca_tree_bits(const uint8_t *row, int S) {
    if (!row) return 0;
    uint64_t bits = 0;
    if (S < 4) {
        for (int j = 0; j < S; ++j) bits |= (uint64_t)(row[j] != 0) << j;
        return bits;
    }
    uint32_t w[CA_MAX_S / 4];
#pragma unroll
    for (int i = 0; i < CA_MAX_S / 4; ++i) {
        w[i] = 0;
        if (4 * i < S) __builtin_memcpy(&w[i], row + (4 * i + 4 <= S ? 4 * i : S - 4), 4);
    }
#pragma unroll
    for (int i = 0; i < CA_MAX_S / 4; ++i) {
        // The bytes that are not 0, as 1 in each, to 4 bits.
        const uint32_t ones = ((((w[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[i]) >> 7) & 0x01010101u;
        const uint32_t four = (ones * 0x01020408u) >> 24;
        bits |= (uint64_t)four << (4 * i + 4 <= S ? 4 * i : S - 4 > 0 ? S - 4 : 0);
    }
    return bits;
}

// The 32 keys from k0 as bits, for the row whose tree bits are `bits`: keys before
// the tree's (from tree0 > k0 - 32 on) are seen, keys past the last are not.
__device__ __forceinline__ uint32_t ca_seen(int64_t k0, int64_t len, int64_t tree0, uint64_t bits) {
    const int64_t s0 = k0 - tree0, left = len - k0;  // s0 > -32, left >= 1
    uint32_t w = s0 >= 0 ? (uint32_t)(bits >> s0) : ((uint32_t)bits << (uint32_t)-s0) | ((1u << (uint32_t)-s0) - 1u);
    if (left < 32) w &= (1u << (uint32_t)left) - 1u;
    return w;
}

// A key that one row does not see may hold infinities or NaN for another.  Such
// values leave the operand v (0 * NaN is NaN); ind gets 1 where they were, so that
// a product of ind and "seen" finds the rows that do see them.  Any in this lane?
__device__ __forceinline__ bool ca_not_finite(bf16x8_t &v, u32x4_t &ind) {
    u32x4_t w = __builtin_bit_cast(u32x4_t, v);
    bool any = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t lo = (w[e] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u;
        const uint32_t hi = (w[e] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
        ind[e] = (lo | hi) & 0x3f803f80u;
        w[e] &= ~(lo | hi);
        any |= (lo | hi) != 0;
    }
    v = __builtin_bit_cast(bf16x8_t, w);
    return any;
}

// Chunk of this workgroup, and its place among the `wide` workgroups (heads and
// row tiles) of that chunk.  Workgroup ids go to the 8 XCDs round-robin; the `wide`
// of one chunk are given to one XCD: a token's exponents of all heads lie in one
// or two lines (32 heads: 128 bytes), which each L2 would otherwise fetch for its
// few heads.
__device__ __forceinline__ uint32_t ca_group(uint32_t wide, uint32_t &at) {
    const uint32_t q = blockIdx.x >> 3, block = q / wide;
    at = q - block * wide;
    return block * 8 + (blockIdx.x & 7);
}

// Inclusive sums over the wave; every lane takes part.
__device__ __forceinline__ int ca_scan(int x, int lane) {  // inclusive, over the wave
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d, 64);
        x += lane >= d ? y : 0;
    }
    return x;
}
// 32 keys of K and V as loaded: K of lane (key, kg) the 16-code chunks 4j + kg of
// keys key and 16 + key; V of a lane, key 8 it + lane / 8, chunk lane % 8.
struct CaRaw {
    uint4 k[2][2], v[4];
    uint32_t ks[2], vs[4];
};

// Keys of one sequence and head: the wave's bases, rows of them in memory, bytes between keys, how many count.
struct CaKeys {
    const uint8_t *kc, *ks, *vc, *vs;
    int64_t C, W, len;
};

// One wave: blocks [blk0, blk1) of 32 keys for 16 * NR query rows, a row per lane % 16.  rows(t, bits) gives the
// address of this lane's row t of q and its tree bits; tree0 is the first key that needs a look at them; vt is the
// wave's V tile.  Returns o (unnormalised, relative to m), the running maximum m and the lane's own share of the sum l.
template <int NR, class Rows>
__device__ __forceinline__ void ca_wave(const CaKeys &k, int64_t blk0, int64_t blk1, float c, int64_t tree0, uint8_t *const vt, Rows rows,
                                        f32x4_t (&o)[NR][8], float (&m)[NR], float (&l)[NR]) {
    const int lane = threadIdx.x & 63, lr = lane & 15, kg = lane >> 4;
    const int64_t len = k.len;
    const float ninf = -__builtin_inff();

    // A block's loads: wave-uniform bases and per-lane 32-bit offsets.  Only a block
    // that reaches past the cache's end clamps its rows to the last one.  The next
    // block's are issued as soon as this one's registers have been consumed.
    const uint8_t *const kc = k.kc, *const vc = k.vc, *const ks = k.ks, *const vs = k.vs;
    const int64_t W = k.W;
    const uint32_t w32 = (uint32_t)W, ws = (uint32_t)(W / 32);
    CaRaw cur;
    auto load_k = [&](int64_t blk) {
        const int64_t k0 = blk * CA_KB;
        const uint8_t *kb = kc + k0 * W, *ksb = ks + k0 * (W / 32);
        const int last = k.C - k0 < CA_KB ? (int)(k.C - k0) - 1 : CA_KB - 1;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t key = 16 * u + lr < last ? 16 * u + lr : last, ko = key * w32 + 16 * kg;
#pragma unroll
            for (int j = 0; j < 2; ++j) cur.k[u][j] = *reinterpret_cast<const uint4 *>(kb + ko + 64 * j);
            cur.ks[u] = *reinterpret_cast<const uint32_t *>(ksb + key * ws);
        }
    };
    auto load_v = [&](int64_t blk) {
        const int64_t k0 = blk * CA_KB;
        const uint8_t *vb = vc + k0 * W, *vsb = vs + k0 * (W / 32);
        const int last = k.C - k0 < CA_KB ? (int)(k.C - k0) - 1 : CA_KB - 1;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const uint32_t vk = 8 * it + (lane >> 3) < last ? 8 * it + (lane >> 3) : last;
            cur.v[it] = *reinterpret_cast<const uint4 *>(vb + (vk * w32 + (lane & 7) * 16));
            cur.vs[it] = vsb[vk * ws + ((lane & 7) >> 1)];
        }
    };
    if (blk0 < blk1) {
        load_v(blk0);
        load_k(blk0);
    }

    // Q operands (step 2j + half: d [64j + 16kg + 8half, +8)) and the tree's bits of
    // this lane's rows.
    bf16x8_t qf[NR][4];
    uint64_t bits[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        const uint16_t *qr = rows(t, bits[t]) + 16 * kg;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            qf[t][2 * j] = *reinterpret_cast<const bf16x8_t *>(qr + 64 * j);
            qf[t][2 * j + 1] = *reinterpret_cast<const bf16x8_t *>(qr + 64 * j + 8);
        }
    }
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        m[t] = ninf;
        l[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[t][dt] = f32x4_t{};
    }

    // This wave's V tile: row = key, 32-byte unit n of key r at unit n ^ (r % 8).
    // Reads: lane i of a 16-lane group addresses 8 bytes of key 4kg + i / 4 (and 16
    // keys later), d 16dt + 4 (i % 4), and receives column i of that 4 x 16 block.
    const uint32_t vbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)vt;
    const int vkey = 4 * kg + (lr >> 2);
    const uint32_t vrow = vbase + vkey * 256 + (lr & 3) * 8;

    for (int64_t blk = blk0; blk < blk1; ++blk) {
        const int64_t k0 = blk * CA_KB;
        const bool whole = k0 + CA_KB <= len;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const int key = 8 * it + (lane >> 3);
            uint4 x = cur.v[it];
            uint32_t e = cur.vs[it];
            if (!whole) {  // V rows past the last key are zeros, whatever the cache holds there
                const bool in = k0 + key < len;
                x = make_uint4(in ? x.x : 0, in ? x.y : 0, in ? x.z : 0, in ? x.w : 0);
                e = in ? e : 0;
            }
            const float sc = mx_scale_operand((int)e);
            uint8_t *at = vt + key * 256 + (((lane & 7) ^ (key & 7)) << 5);
            *reinterpret_cast<bf16x8_t *>(at) = ca_operand(x.x, x.y, sc);
            *reinterpret_cast<bf16x8_t *>(at + 16) = ca_operand(x.z, x.w, sc);
        }
        if (blk + 1 < blk1) load_v(blk + 1);
        f32x4_t s[NR][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float sc = mx_scale_operand((int)((cur.ks[u] >> (8 * (2 * j + (kg >> 1)))) & 0xffu));
                const uint4 x = cur.k[u][j];
                const bf16x8_t k_lo = ca_operand(x.x, x.y, sc), k_hi = ca_operand(x.z, x.w, sc);
#pragma unroll
                for (int t = 0; t < NR; ++t) {
                    s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k_lo, qf[t][2 * j], j == 0 ? f32x4_t{} : s[t][u], 0, 0, 0);
                    s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k_hi, qf[t][2 * j + 1], s[t][u], 0, 0, 0);
                }
            }
        if (blk + 1 < blk1) load_k(blk + 1);
        // Only blocks that reach the tree's keys or the end have anything masked.
        const bool masked = k0 + CA_KB > tree0;
        uint32_t seen[NR];
        u32x4_t pw[NR], pl[NR];
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            seen[t] = ~0u;
            if (masked) {
                seen[t] = ca_seen(k0, len, tree0, bits[t]) >> (4 * kg);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][u][i] = (seen[t] >> (16 * u + i)) & 1u ? s[t][u][i] : ninf;
            }
            float mx = ca_max(ca_max(ca_max(s[t][0][0], s[t][0][1]), ca_max(s[t][0][2], s[t][0][3])),
                              ca_max(ca_max(s[t][1][0], s[t][1][1]), ca_max(s[t][1][2], s[t][1][3])));
            {
                const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
                mx = ca_swap_max(ca_max(__uint_as_float(sw[0]), __uint_as_float(sw[1]))) * c;
            }
            const float mn = ca_max(m[t], mx);
            const float ref = mn == ninf ? 0.f : mn;  // nothing seen yet: every p is 0
            const float alpha = __builtin_amdgcn_exp2f(m[t] - ref);
            m[t] = mn;
            float e[8], sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i >> 2][i & 3], c, -ref));
                sum += e[i];
            }
            l[t] = l[t] * alpha + sum;
            // p enters the matrix product as two bf16 terms, pw + pl (pl the rounding
            // error of pw): 16 significand bits, where pw alone would put 2^-8 of each
            // term into the sum while l keeps all of it.
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                pw[t][i] = pack_bf16x2(e[2 * i], e[2 * i + 1]);
                pl[t][i] = pack_bf16x2(e[2 * i] - bf_lo(pw[t][i]), e[2 * i + 1] - bf_hi(pw[t][i]));
            }
            if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) o[t][dt] *= alpha;
            }
        }
        // A wave's LDS operations run in order; the compiler must not reorder them.
        asm volatile("" ::: "memory");
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            typedef __attribute__((address_space(3))) i16x4_t *ptr_t;
            const uint32_t at = vrow + ((dt ^ (vkey & 7)) << 5);
            const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<ptr_t>((uintptr_t)at));
            const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<ptr_t>((uintptr_t)(at + 16 * CA_D * 2)));
            bf16x8_t vf = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            if (masked) {
                u32x4_t ind;
                if (__builtin_amdgcn_ballot_w64(ca_not_finite(vf, ind))) {
#pragma unroll
                    for (int t = 0; t < NR; ++t) {
                        u32x4_t sv;
#pragma unroll
                        for (int e2 = 0; e2 < 4; ++e2) {
                            const uint32_t two = seen[t] >> (16 * (e2 >> 1) + 2 * (e2 & 1));
                            sv[e2] = ((two & 1u) ? 0x3f80u : 0u) | ((two & 2u) ? 0x3f800000u : 0u);
                        }
                        const f32x4_t hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            __builtin_bit_cast(bf16x8_t, ind), __builtin_bit_cast(bf16x8_t, sv), f32x4_t{}, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[t][dt][i] = hit[i] > 0.f ? __builtin_nanf("") : o[t][dt][i];
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NR; ++t) {
                o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8_t, pl[t]), o[t][dt], 0, 0, 0);
                o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8_t, pw[t]), o[t][dt], 0, 0, 0);
            }
        }
        asm volatile("" ::: "memory");
    }
}

}  // namespace qim
