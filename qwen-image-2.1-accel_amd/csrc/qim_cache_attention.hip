// Attention of a few tokens over a K/V cache in MXFP8 (qim_cache.hip): one
// token of each request, or up to 64 drafted ones with a tree mask, head dim
// 128, query heads in groups of G that share a K/V head.
//
//   o[r] = sum_t p_rt V[t] / sum_t p_rt,  p_rt = 2^(c q_r . K[t] - m_r)
//
// in one pass over the keys with a running maximum m_r and sum (fp32).  The
// S * G query rows that share a K/V head are the columns of the MFMA tiles, 16 or 32
// to a wave.  A row costs 512 flop for a key's 264 bytes: up to 32 rows the cache's
// bytes bound it, more rows the waves' work on codes and softmax.
//
// Transposed products on v_mfma_f32_16x16x32_bf16, 32 keys at a time: S^T = K Q^T
// (two tiles of 16 keys x 16 rows) and O^T = V^T P^T (16 head dims x 16 rows per
// tile), so a lane owns query row lane % 16 in both; with kg = lane / 16 its scores
// are those of keys 16u + 4kg + i (u = 0, 1; i = 0..3), which is its B operand of one
// 32-key step of the second product, and a row's maximum is one value exchanged
// between 4 lanes per block.  Codes become bf16 exactly (4 significand bits times
// a power of two), the block's exponent being the conversion's scale operand.  K goes
// from memory to the A operand as it is: a 16-code chunk is two 8-value operands,
// and Q is held in the same order (an MFMA pairs the K slots of A and B by
// position).  V is converted into a per-wave LDS tile of 32 keys x 128 and
// transposed by the LDS reads.
//
// Where there are too few (sequence, head) pairs to fill the chip, or their keys are
// many, the keys are cut into chunks and a second launch joins them.
//
// One row a head: 16 sequences of up to 8392 keys, 32 heads, 168 us (869 MB, 5.2 TB/s); 2 of
// up to 131072 with 8 K/V heads of 4 rows 88 us (484 MB, 5.5 TB/s); the join 5 us.  24 rows a
// head, 4 sequences of up to 8392 keys: 59 us (3.9 TB/s); the join of 24 MB 6.2 us.
// The second term of p costs 0.9 us of these 59, nothing with one row a head.
#include "qim_device.h"
#include "qim_runtime.h"

namespace qim {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

constexpr int CA_D = 128;
constexpr int CA_KB = 32;                        // keys per block
constexpr int CA_VTILE = CA_KB * CA_D * 2;       // 8 KiB of LDS per wave
constexpr int CA_WAVES = 8;                      // (heads) per workgroup: two per SIMD
constexpr int CA_MAX_S = 64;
constexpr int CA_MAX_ROUNDS = 16;

struct CacheAttnArgs {
    const uint16_t *q;
    int64_t ldqb, ldq;
    const uint8_t *kc, *ks, *vc, *vs;
    const int32_t *lengths;
    const uint8_t *tree;
    int64_t tree_b;
    uint16_t *o;
    float *part_o;   // (chunk, K/V head, row, 128), relative to the chunk's maximum
    float2 *part_ml; // (chunk, K/V head, row): (maximum, sum)
    int64_t C;
    int2 *dir;       // per sequence: its first chunk and their number
    int B, S, H, HK, G, rows, ntile;
    int chunks;      // key chunks over all sequences, short of one per sequence; 0: a sequence is one chunk, nothing to join
    float scale_log2e;
};

// The bf16 operand of 8 codes of a block.
__device__ __forceinline__ bf16x8_t ca_operand(uint32_t lo, uint32_t hi, float scale) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ int64_t ca_length(const CacheAttnArgs &p, int64_t b) {
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : n > p.C ? p.C : n;
}
__device__ __forceinline__ float ca_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float ca_swap_max(float x) {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return ca_max(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

// The tree's bits of query s: bit j, whether it sees the j-th of the last S keys.
// Four truth bytes per load (rows of S bytes, any alignment), all loads in flight
// together; the last load ends at the row's end and repeats bits.
__device__ __forceinline__ uint64_t ca_tree_bits(const CacheAttnArgs &p, int b, int s) {
    if (!p.tree) return 0;
    const uint8_t *row = p.tree + b * p.tree_b + s * p.S;
    uint64_t bits = 0;
    if (p.S < 4) {
        for (int j = 0; j < p.S; ++j) bits |= (uint64_t)(row[j] != 0) << j;
        return bits;
    }
    uint32_t w[CA_MAX_S / 4];
#pragma unroll
    for (int i = 0; i < CA_MAX_S / 4; ++i) {
        w[i] = 0;
        if (4 * i < p.S) __builtin_memcpy(&w[i], row + (4 * i + 4 <= p.S ? 4 * i : p.S - 4), 4);
    }
#pragma unroll
    for (int i = 0; i < CA_MAX_S / 4; ++i) {
        // The bytes that are not 0, as 1 in each, to 4 bits.
        const uint32_t ones = ((((w[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[i]) >> 7) & 0x01010101u;
        const uint32_t four = (ones * 0x01020408u) >> 24;
        bits |= (uint64_t)four << (4 * i + 4 <= p.S ? 4 * i : p.S - 4 > 0 ? p.S - 4 : 0);
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

// The chunks: all sequences' blocks of 32 keys, whatever their lengths, are cut into
// pieces of `per` blocks, the smallest of which there are at most p.chunks + B (a
// sequence's last piece may be shorter): equal shares for the waves in a batch of
// unequal lengths, and never a few workgroups more than fit.  Finds sequence and
// piece of chunk `group`; false past the last.  The first workgroup also writes
// p.dir for the join.  Every lane of the wave takes part.
__device__ __forceinline__ int ca_scan(int x, int lane) {  // inclusive, over the wave
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d, 64);
        x += lane >= d ? y : 0;
    }
    return x;
}
__device__ __forceinline__ bool ca_chunk(const CacheAttnArgs &p, uint32_t group, bool writes, int &b, int64_t &blk0, int64_t &per) {
    if (!p.chunks) {
        b = (int)group;
        blk0 = 0;
        per = p.C;
        return b < p.B;
    }
    const int lane = threadIdx.x & 63;
    auto blocks = [&](int i) { return i < p.B ? (int)((ca_length(p, i) + CA_KB - 1) / CA_KB) : 0; };
    int64_t total = 0;
    for (int i = 0; i < p.B; i += 64) total += __builtin_amdgcn_readlane(ca_scan(blocks(i + lane), lane), 63);
    const int each = (int)((total + p.chunks - 1) / p.chunks);
    per = each > 1 ? each : 1;
    uint32_t first = 0;
    bool found = false;
    for (int i = 0; i < p.B && !(found && !writes); i += 64) {
        const int n = (blocks(i + lane) + (int)per - 1) / (int)per, last = ca_scan(n, lane);
        const uint32_t from = first + last - n;
        if (writes && i + lane < p.B) p.dir[i + lane] = make_int2((int)from, n);
        const uint64_t here = __builtin_amdgcn_ballot_w64(group >= from && group < from + n);
        if (here) {
            const int at = (int)__builtin_ctzll(here);
            b = i + at;
            blk0 = (int64_t)(group - (uint32_t)__builtin_amdgcn_readlane((int)from, at)) * per;
            found = true;
        }
        first += (uint32_t)__builtin_amdgcn_readlane(last, 63);
    }
    return found;
}

// 32 keys of K and V as loaded: K of lane (key, kg) the 16-code chunks 4j + kg of
// keys key and 16 + key; V of a lane, key 8 it + lane / 8, chunk lane % 8.
struct CaRaw {
    uint4 k[2][2], v[4];
    uint32_t ks[2], vs[4];
};

// One wave: a (sequence, K/V head, tile of 16 * NR rows, key chunk) of its own;
// neighbouring waves take neighbouring heads, whose 128-byte pieces are neighbours in
// memory.  No barrier anywhere.
template <int NR>
__global__ __launch_bounds__(64 * CA_WAVES, 2) void k_cache_attn(CacheAttnArgs p) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[CA_WAVES * CA_VTILE];
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t tasks = (uint32_t)(p.HK * p.ntile);
    uint32_t task;
    const uint32_t group = ca_group((tasks + CA_WAVES - 1) / CA_WAVES, task);
    int b = 0;
    int64_t blk0 = 0, per = 1;
    if (!ca_chunk(p, group, blockIdx.x == 0 && wave == 0, b, blk0, per)) return;
    task = task * CA_WAVES + wave;
    if (task >= tasks) return;
    const int tile = (int)(task / (uint32_t)p.HK), h = (int)(task - tile * (uint32_t)p.HK);
    const int64_t len = ca_length(p, b);
    const int64_t nblk = (len + CA_KB - 1) / CA_KB, blk1 = blk0 + per < nblk ? blk0 + per : nblk;
    const float c = p.scale_log2e, ninf = -__builtin_inff();

    // A block's loads: wave-uniform bases and per-lane 32-bit offsets.  Only a block
    // that reaches past the cache's end clamps its rows to the last one.  The next
    // block's are issued as soon as this one's registers have been consumed.
    const int64_t W = (int64_t)p.HK * CA_D;
    const uint8_t *kc = p.kc + b * p.C * W + h * CA_D, *vc = p.vc + b * p.C * W + h * CA_D;
    const uint8_t *ks = p.ks + (b * p.C * W + h * CA_D) / 32, *vs = p.vs + (b * p.C * W + h * CA_D) / 32;
    const uint32_t w32 = (uint32_t)W, ws = (uint32_t)(W / 32);
    CaRaw cur;
    auto load_k = [&](int64_t blk) {
        const int64_t k0 = blk * CA_KB;
        const uint8_t *kb = kc + k0 * W, *ksb = ks + k0 * (W / 32);
        const int last = p.C - k0 < CA_KB ? (int)(p.C - k0) - 1 : CA_KB - 1;
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
        const int last = p.C - k0 < CA_KB ? (int)(p.C - k0) - 1 : CA_KB - 1;
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
    int row[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        row[t] = (tile * NR + t) * 16 + lr;
        const int r = row[t] < p.rows ? row[t] : p.rows - 1;  // rows past the end: computed, not stored
        const int s = r / p.G, head = h * p.G + (r - s * p.G);
        const uint16_t *qr = p.q + b * p.ldqb + s * p.ldq + head * CA_D + 16 * kg;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            qf[t][2 * j] = *reinterpret_cast<const bf16x8_t *>(qr + 64 * j);
            qf[t][2 * j + 1] = *reinterpret_cast<const bf16x8_t *>(qr + 64 * j + 8);
        }
        bits[t] = ca_tree_bits(p, b, s);
    }
    f32x4_t o[NR][8];
    float m[NR], l[NR];
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
    uint8_t *const vt = lds + wave * CA_VTILE;
    const uint32_t vbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)vt;
    const int vkey = 4 * kg + (lr >> 2);
    const uint32_t vrow = vbase + vkey * 256 + (lr & 3) * 8;
    const int64_t tree0 = p.tree ? len - p.S : len;  // the first key that needs a look at the mask

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
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        float lt = l[t] + __shfl_xor(l[t], 16, 64);
        lt += __shfl_xor(lt, 32, 64);
        if (row[t] >= p.rows) continue;
        if (!p.chunks) {
            const float inv = lt == 0.f ? 0.f : 1.0f / lt;  // no visible key: zeros
            const int s = row[t] / p.G, head = h * p.G + (row[t] - s * p.G);
            uint16_t *dst = p.o + (((int64_t)b * p.S + s) * p.H + head) * CA_D + 4 * kg;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt)
                *reinterpret_cast<uint2 *>(dst + 16 * dt) = make_uint2(pack_bf16x2(o[t][dt][0] * inv, o[t][dt][1] * inv),
                                                                       pack_bf16x2(o[t][dt][2] * inv, o[t][dt][3] * inv));
        } else {
            const int64_t at = ((int64_t)group * p.HK + h) * p.rows + row[t];
            float *dst = p.part_o + at * CA_D + 4 * kg;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4_t *>(dst + 16 * dt) = o[t][dt];
            if (kg == 0) p.part_ml[at] = make_float2(m[t], lt);
        }
    }
}

// Join the key chunks of a row: GP groups of LANES lanes (4 head dims each) take the
// chunks of 4 * LANES head dims in turn, four loads at a time, and join in LDS.
template <int GP, int LANES>
__global__ __launch_bounds__(256) void k_cache_attn_join(CacheAttnArgs p, int64_t nparts) {
    constexpr int PARTS = 32 / LANES, NG = 256 / LANES;  // parts of a row; groups of the workgroup
    __shared__ float4 so[NG][LANES];
    __shared__ float2 sml[NG];
    const int grp = threadIdx.x / LANES, ln = threadIdx.x % LANES;
    const int64_t g = (int64_t)blockIdx.x * (NG / GP) + grp / GP;
    const bool live = g < nparts;
    const int64_t row = live ? g / PARTS : 0, item0 = row / p.rows;  // (sequence, K/V head)
    const int d0 = (int)(g % PARTS) * (4 * LANES) + ln * 4;
    const int r = (int)(row - item0 * p.rows);
    const int64_t b = item0 / p.HK;
    const int2 dir = p.dir[b];
    const int n = dir.y;  // chunks of this sequence
    const int64_t step = (int64_t)p.HK * p.rows, first = dir.x * step + (item0 - b * p.HK) * p.rows + r;
    const float ninf = -__builtin_inff();
    float M = ninf, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = grp % GP; i < n; i += 4 * GP) {
        float2 ml[4];
        float4 f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t at = first + (i + j * GP < n ? i + j * GP : i) * step;
            ml[j] = p.part_ml[at];
            f[j] = *reinterpret_cast<const float4 *>(p.part_o + at * CA_D + d0);
            if (i + j * GP >= n) ml[j] = make_float2(ninf, 0.f);
        }
        float Mn = M;
#pragma unroll
        for (int j = 0; j < 4; ++j) Mn = ca_max(Mn, ml[j].x);
        const float ref = Mn == ninf ? 0.f : Mn, sc = __builtin_amdgcn_exp2f(M - ref);
        L *= sc;
        acc = make_float4(acc.x * sc, acc.y * sc, acc.z * sc, acc.w * sc);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float w = __builtin_amdgcn_exp2f(ml[j].x - ref);
            if (i + j * GP < n) {  // (a repeated chunk may hold NaN)
                L += ml[j].y * w;
                acc = make_float4(acc.x + f[j].x * w, acc.y + f[j].y * w, acc.z + f[j].z * w, acc.w + f[j].w * w);
            }
        }
        M = Mn;
    }
    if constexpr (GP > 1) {
        so[grp][ln] = acc;
        if (ln == 0) sml[grp] = make_float2(M, L);
        __syncthreads();
        if (grp % GP) return;
        M = ninf;
#pragma unroll
        for (int j = 0; j < GP; ++j) M = ca_max(M, sml[grp + j].x);
        const float ref = M == ninf ? 0.f : M;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
        L = 0.f;
#pragma unroll
        for (int j = 0; j < GP; ++j) {
            const float w = __builtin_amdgcn_exp2f(sml[grp + j].x - ref);
            const float4 f = so[grp + j][ln];
            L += sml[grp + j].y * w;
            acc = make_float4(acc.x + f.x * w, acc.y + f.y * w, acc.z + f.z * w, acc.w + f.w * w);
        }
    }
    if (!live) return;
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    const int h = (int)(item0 % p.HK), s = r / p.G, head = h * p.G + (r - s * p.G);
    uint16_t *dst = p.o + ((b * p.S + s) * p.H + head) * CA_D + d0;
    *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

// Row tiles (16 or 32 rows a wave) and key chunks.  A chunk's heads and row tiles are
// `wide` workgroups of one XCD, one workgroup to a CU, so `cap` chunks run at a time;
// the chunks are to fill whole rounds.  What is weighed, in ns: a block of 32 keys
// costs a round the time of its bytes, or that of a wave's work where rows share them
// (8 waves a CU: 2100 with 16 rows, 3000 with 32); a round 1500 for its start;
// chunks 5000 for the second launch and their partial results, written and read.
// (With the join, 5 sequences of up to 8040 keys, 64 rows a head, 32 heads: 196 us as 16
// rows a wave, 136 as 32; 14 of up to 428: 41 and 52.  64 rows a wave gained nothing:
// 128 and 53 where 32 took 118 and 48, without the join and p's second term.  16 of up to 8392, one row: 5 rounds of chunks 168 us, 2.95 172, 2.1 200; 2 of up to
// 131072, 8 heads: 249 chunks 88 us, 257 chunks 119.)
struct CaPlan {
    int64_t rows, nr, ntile, wide, chunks, groups, B, HK;
    int64_t grid() const { return (groups + 7) / 8 * 8 * wide; }  // ca_group
    int64_t part_o() const { return chunks ? groups * HK * rows * CA_D * 4 : 0; }
    int64_t part_ml() const { return chunks ? groups * HK * rows * 8 : 0; }
    int64_t bytes() const { return chunks ? part_o() + part_ml() + B * 8 : 0; }
};
static CaPlan ca_plan(int64_t B, int64_t S, int64_t C, int64_t H, int64_t HK) {
    CaPlan pl;
    pl.B = B;
    pl.HK = HK;
    pl.rows = S * (H / HK);
    const int64_t cus = device_cus() > 0 ? device_cus() : 256, nblk = (C + CA_KB - 1) / CA_KB;
    int64_t best = -1;
    for (int64_t nr = 1; nr <= 2 && (nr - 1) * 16 < pl.rows; ++nr) {
        const int64_t ntile = (pl.rows + 16 * nr - 1) / (16 * nr), wide = (HK * ntile + CA_WAVES - 1) / CA_WAVES;
        const int64_t at_once = cus / 8 / wide, cap = 8 * (at_once > 1 ? at_once : 1);
        // r rounds of chunks; 0: a chunk per sequence and nothing to join.
        for (int64_t r = 0; r <= CA_MAX_ROUNDS && (r == 0 || nblk > 1); ++r) {
            const int64_t n = r * cap - B;
            if (r && n < 1) continue;
            const int64_t groups = r == 0 ? B : n + B < B * nblk ? n + B : B * nblk;
            const int64_t rounds = r ? r : (B + cap - 1) / cap, blocks = r ? (B * nblk + n - 1) / n : nblk;
            const int64_t bytes = (groups < cap ? groups : cap) * HK * CA_KB * 2 * (CA_D + CA_D / 32);
            const int64_t work = nr == 1 ? 2100 : 3000, block = bytes / 5140 > work ? bytes / 5140 : work;
            const int64_t cost = rounds * (blocks * block + 1500) + (r ? 5000 + groups * HK * pl.rows * CA_D * 8 / 5140 : 0);
            if (best >= 0 && cost >= best) continue;
            best = cost;
            pl.nr = nr;
            pl.ntile = ntile;
            pl.wide = wide;
            pl.chunks = r ? n : 0;
            pl.groups = groups;
        }
    }
    return pl;
}

}  // namespace qim

using namespace qim;

static bool ca_shape(int64_t B, int64_t S, int64_t C, int64_t H, int64_t HK) {
    return B > 0 && S > 0 && S <= CA_MAX_S && C > 0 && C < (1ll << 31) && HK > 0 && H > 0 && H % HK == 0 && H <= (1 << 16) && B < (1 << 20) &&
           B * HK * ((S * (H / HK) + 15) / 16) < (1 << 25) && B * C < (1ll << 40) / HK && ca_plan(B, S, C, H, HK).grid() * (64 * CA_WAVES) < (1ll << 32);
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
    // Rows are written while others are still read.
    const char *q0 = (const char *)q, *q1 = q0 + 2 * ((B - 1) * ldqb + (S - 1) * ldq + H * D), *o0 = (const char *)o;
    QIM_REQUIRE(q1 <= o0 || o0 + 2 * B * S * H * D <= q0, QIM_ERR_ARG, "%s: o overlaps q", who);
    void (*const fn)(CacheAttnArgs) = pl.nr == 1 ? k_cache_attn<1> : k_cache_attn<2>;
    uint8_t *const ws = static_cast<uint8_t *>(workspace);
    CacheAttnArgs a{(const uint16_t *)q, ldqb, ldq, (const uint8_t *)kc, (const uint8_t *)ks, (const uint8_t *)vc,
                    (const uint8_t *)vs, lengths, (const uint8_t *)tree, tree_b, (uint16_t *)o, (float *)ws,
                    (float2 *)(ws + pl.part_o()), C, (int2 *)(ws + pl.part_o() + pl.part_ml()), (int)B, (int)S, (int)H,
                    (int)HK, (int)(H / HK), (int)pl.rows, (int)pl.ntile, (int)pl.chunks,
                    scale * 1.4426950408889634f};
    launch(fn, dim3((unsigned)pl.grid()), dim3(64 * CA_WAVES), 0, as_stream(stream), a);
    if (pl.chunks) {
        // Few rows of many chunks: a quarter row per workgroup, 32 chunks at once.
        const int64_t nrows = B * HK * pl.rows, each = pl.groups / B;
        const bool many = each > 16 && 2 * nrows <= device_cus();
        const int64_t gp = each > 16 ? 8 : each > 4 ? 2 : 1;
        launch(many ? k_cache_attn_join<32, 8> : gp == 8 ? k_cache_attn_join<8, 32> : gp == 2 ? k_cache_attn_join<2, 32> : k_cache_attn_join<1, 32>,
               dim3((unsigned)(many ? nrows * 4 : (nrows * gp + 7) / 8)), dim3(256), 0, as_stream(stream), a, many ? nrows * 4 : nrows);
    }
    return check_launch(who);
}
