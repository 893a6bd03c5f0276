// Attention of a few tokens of many requests that continue shared prefixes: the prefixes and the requests' own keys in
// MXFP8 caches (qim_cache.hip), head dim 128, query heads in groups of G that share a K/V head.
//
//   o[r] = (sum_prefix p_t V[t] + sum_own p_t V[t]) / (sum_prefix p_t + sum_own p_t),  p_t = 2^(c q_r . K[t] - m_r)
//
// The rows of all requests on one prefix (requests * S * G to a K/V head) are the columns of the same matrix products, so
// that a prefix's codes are read and converted once for a tile of rows instead of once for every request.  Prefix and own
// keys give partial results (numerator, maximum, sum; fp32) over chunks of keys, joined in a last launch.
//
// Few rows: the cache's bytes and the launches' starts bound it; from some 64 rows on the vector instructions of the softmax and
// the conversions, beside the matrix products.  Measured (launches from a graph): 4 requests, one row each on 32 heads, 1101 +
// 96 keys 13.2 us (8.6 and the join's 4.9); 32 requests of 4 rows on 8 heads, 8392 + 1024 keys 30 us; 48 requests on 5
// prefixes of up to 32768 keys 86 us, 3.6 TB/s; 8 requests of 24 rows on 32 heads, 8392 + 256 keys 71-74 us, 370 TFLOP/s.
//
// The rows of a prefix: its requests in the order of their numbers, S * G rows each.  Which requests those are is known on
// the device only.  Up to 64 requests and 16 prefixes every wave finds them itself, a request a lane (48 requests on 5
// prefixes 3 us less than with a launch for it); of more, a first launch of one workgroup makes lists.  It looks at every
// request for every prefix: 65 requests on 17 prefixes 3.6 us, 256 on 64 8.7, 1024 on 64 30, 1024 on 512 164, 4096 on 1024 1168,
// which from some 512 prefixes on is as long as the attention itself (8 K/V heads, short prefixes).
#include "qim_cache_attention.h"
#include "qim_runtime.h"

namespace qim {

constexpr int SA_WAVES = 4;
constexpr int SA_MAX_PREFIXES = 4096;
constexpr int SA_FEW_PREFIXES = 16;

// A space of keys: V sequences (own: a request and a tile of its rows; prefix: a tile of rows) cut into at most `most` pieces
// (V or more).  Partial results by (piece, K/V head, row of the tile).
struct SaSpace {
    float *part_o;    // 128 values each
    float2 *part_ml;  // (maximum, sum)
    int2 *dir;        // per sequence: its first piece and their number
    int V, most, rows;
    int keys;         // of a block: pieces are whole blocks
    uint32_t blocks;  // workgroups
};
struct SaArgs {
    const uint16_t *q;
    int64_t ldqb, ldq;
    const uint8_t *pk, *pks, *pv, *pvs, *kc, *ks, *vc, *vs;
    const int32_t *lengths, *plengths, *share;
    const uint8_t *tree;
    int64_t tree_b, CP, C;
    uint16_t *o;
    SaSpace pre, own;
    int few;          // share: no lists, every wave has a request and a prefix tile a lane
    int4 *tiles;      // per prefix tile: prefix, first of its requests in `order`, their rows, the tile's first row (share only)
    int32_t *order;   // the requests by prefix
    int2 *where;      // per request: its prefix's first tile (-1: none), its place among the prefix's requests
    int B, S, H, HK, G, P, ntile;  // ntile: row tiles of a request's own keys
    float scale_log2e;
};

__device__ __forceinline__ int64_t sa_clamp(int64_t n, int64_t most) { return n < 0 ? 0 : n > most ? most : n; }
__device__ __forceinline__ int64_t sa_prefix_length(const SaArgs &p, int i) { return p.plengths ? sa_clamp(p.plengths[i], p.CP) : p.CP; }

// Rows of a prefix tile.
struct SaTile {
    int prefix, first, rows, row0;
};
__device__ __forceinline__ SaTile sa_tile(const SaArgs &p, int i) {
    if (!p.share) return SaTile{0, 0, p.B * p.S * p.G, i * p.pre.rows};
    const int4 t = p.tiles[i];
    return SaTile{t.x, t.y, t.z, t.w};
}

// What a lane holds of the plan where the batch is small: its request's prefix, and the prefix tile of its number.
struct SaLanes {
    int who;
    SaTile tile;
};
template <class Each>
__device__ __forceinline__ void sa_each_prefix(const SaArgs &p, int who, Each each) {  // (prefix, its requests, its first tile, tiles)
    const int shift = __builtin_ctz((unsigned)p.pre.rows);
    int first = 0;
    for (int i = 0; i < p.P; ++i) {
        const uint64_t all = __builtin_amdgcn_ballot_w64(who == i);
        const int tiles = ((int)__builtin_popcountll(all) * p.S * p.G + p.pre.rows - 1) >> shift;
        each(i, all, first, tiles);
        first += tiles;
    }
}
__device__ __forceinline__ SaLanes sa_lanes(const SaArgs &p) {
    const int lane = threadIdx.x & 63;
    SaLanes l{-1, SaTile{0, 0, 0, 0}};
    if (!p.few) return l;
    l.who = lane < p.B ? p.share[lane] : -1;
    sa_each_prefix(p, l.who, [&](int i, uint64_t all, int first, int tiles) {
        if (lane >= first && lane < first + tiles) l.tile = SaTile{i, 0, (int)__builtin_popcountll(all) * p.S * p.G, (lane - first) * p.pre.rows};
    });
    return l;
}
__device__ __forceinline__ SaTile sa_tile(const SaArgs &p, const SaLanes &l, int i) {
    if (!p.few) return sa_tile(p, i);
    return SaTile{__builtin_amdgcn_readlane(l.tile.prefix, i), 0, __builtin_amdgcn_readlane(l.tile.rows, i), __builtin_amdgcn_readlane(l.tile.row0, i)};
}
// The requests of a tile's prefix, one a lane, in their order (few only).
__device__ __forceinline__ int sa_requests(const SaArgs &p, const SaLanes &l, int prefix) {
    if (!p.few) return 0;
    const int lane = threadIdx.x & 63;
    const uint64_t all = __builtin_amdgcn_ballot_w64(l.who == prefix), below = (1ull << lane) - 1;
    const int at = l.who == prefix ? (int)__builtin_popcountll(all & below) : (int)(__builtin_popcountll(all) + __builtin_popcountll(~all & below));
    return __builtin_amdgcn_ds_permute(4 * at, lane);
}
__device__ __forceinline__ int sa_request(const SaArgs &p, const SaTile &t, int requests, int i) {
    if (!p.share) return i;
    return p.few ? __shfl(requests, i, 64) : p.order[t.first + i];
}

// The requests of each prefix, in their order, and the prefix's tiles of rows.  One workgroup; a wave per prefix counts and
// lists with ballots, 64 requests at a time.
__global__ __launch_bounds__(1024) void k_shared_plan(SaArgs p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    int32_t *const first = reinterpret_cast<int32_t *>(lds), *const tile = first + p.P;  // of each prefix: count, then first request; first tile
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = wave; i < p.P; i += 16) {
        int n = 0;
        for (int b = 0; b < p.B; b += 64)
            n += (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(b + lane < p.B && p.share[b + lane] == i));
        if (lane == 0) first[i] = n;
    }
    __syncthreads();
    if (wave == 0) {
        int requests = 0, tiles = 0;
        for (int i = 0; i < p.P; i += 64) {
            const int n = i + lane < p.P ? first[i + lane] : 0, t = (n * p.S * p.G + p.pre.rows - 1) / p.pre.rows;
            const int ns = ca_scan(n, lane), ts = ca_scan(t, lane);
            if (i + lane < p.P) {
                first[i + lane] = requests + ns - n;
                tile[i + lane] = tiles + ts - t;
            }
            requests += __builtin_amdgcn_readlane(ns, 63);
            tiles += __builtin_amdgcn_readlane(ts, 63);
        }
        // Tiles that no prefix needs hold no rows.
        for (int i = tiles + lane; i < p.pre.V; i += 64) p.tiles[i] = make_int4(0, 0, 0, 0);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < p.B; b += 1024)
        if (p.share[b] < 0 || p.share[b] >= p.P) p.where[b] = make_int2(-1, 0);
    for (int i = wave; i < p.P; i += 16) {
        int n = 0;
        for (int b = 0; b < p.B; b += 64) {
            const bool mine = b + lane < p.B && p.share[b + lane] == i;
            const uint64_t all = __builtin_amdgcn_ballot_w64(mine);
            if (mine) {
                const int at = n + (int)__builtin_popcountll(all & ((1ull << lane) - 1));
                p.order[first[i] + at] = b + lane;
                p.where[b + lane] = make_int2(tile[i], at);
            }
            n += (int)__builtin_popcountll(all);
        }
        const int rows = n * p.S * p.G;
        for (int t = lane; t * p.pre.rows < rows; t += 64) p.tiles[tile[i] + t] = make_int4(i, first[i], rows, t * p.pre.rows);
    }
}

template <bool PRE>
__device__ __forceinline__ int64_t sa_length(const SaArgs &p, const SaLanes &l, int i) {  // (few: i is the lane's own number)
    if constexpr (PRE) {
        const SaTile t = p.few ? l.tile : sa_tile(p, i);
        return t.rows ? sa_prefix_length(p, t.prefix) : 0;
    }
    return sa_clamp(p.lengths[i / p.ntile], p.C);
}

// Which piece this is: sequence v, its blocks [blk0, blk0 + per).  All sequences' blocks are cut into pieces of `per`, of
// which there are at most sp.most.  The first workgroup also writes the space's dir.
template <bool PRE>
__device__ __forceinline__ bool sa_piece(const SaArgs &p, const SaLanes &l, const SaSpace &sp, uint32_t piece, bool writes, int &v, int &blk0, int &per) {
    const int lane = threadIdx.x & 63;
    if (PRE && !p.share) {  // sequences alike: the same pieces of each
        const int n = (int)(((uint32_t)sa_prefix_length(p, 0) + sp.keys - 1) / (uint32_t)sp.keys), each = sp.most / sp.V;
        const int size = n > each ? (n + each - 1) / each : 1, count = (n + size - 1) / size;
        per = size;
        if (writes)
            for (int i = lane; i < sp.V; i += 64) sp.dir[i] = make_int2(i * count, count);
        if (!count || piece >= (uint32_t)(sp.V * count)) return false;
        v = (int)(piece / (uint32_t)count);
        blk0 = ((int)piece - v * count) * size;
        return true;
    }
    auto blocks = [&](int i) { return i < sp.V ? (int)(((uint32_t)sa_length<PRE>(p, l, i) + sp.keys - 1) / (uint32_t)sp.keys) : 0; };
    const int head = blocks(lane);  // the first 64 sequences' stay in a register
    auto blocks_from = [&](int i) { return i ? blocks(i + lane) : head; };
    uint32_t total = 0;  // (all spaces have fewer than 2^31 blocks)
    for (int i = 0; i < sp.V; i += 64) total += (uint32_t)__builtin_amdgcn_readlane(ca_scan(blocks_from(i), lane), 63);
    // The smallest `per` that is sure to give at most `most` pieces, or a smaller one that happens to.
    auto pieces = [&](uint32_t of) {
        int n = 0;
        for (int i = 0; i < sp.V; i += 64) n += __builtin_amdgcn_readlane(ca_scan((int)((blocks_from(i) + of - 1) / of), lane), 63);
        return n;
    };
    const int spare = sp.most - sp.V > 1 ? sp.most - sp.V : 1;
    const uint32_t sure = (total + spare - 1) / (uint32_t)spare;
    uint32_t of = (total + sp.most - 1) / (uint32_t)sp.most;
    of = of > 1 ? of : 1;
    while (of < sure && pieces(of) > sp.most) of = of + of / 8 + 1;
    of = of < sure || sure < 1 ? of : sure;
    per = (int)of;
    uint32_t first = 0;
    bool found = false;
    for (int i = 0; i < sp.V && !(found && !writes); i += 64) {
        const int n = (int)((blocks_from(i) + of - 1) / of), last = ca_scan(n, lane);
        const uint32_t from = first + last - n;
        if (writes && i + lane < sp.V) sp.dir[i + lane] = make_int2((int)from, n);
        const uint64_t here = __builtin_amdgcn_ballot_w64(piece >= from && piece < from + n);
        if (here) {
            const int at = (int)__builtin_ctzll(here);
            v = i + at;
            blk0 = (int)(piece - (uint32_t)__builtin_amdgcn_readlane((int)from, at)) * per;
            found = true;
        }
        first += (uint32_t)__builtin_amdgcn_readlane(last, 63);
    }
    return found;
}

// One wave: a piece of keys of one K/V head for a tile of 16 * NR rows.
template <bool PRE, int NR>
__device__ __forceinline__ void sa_wave(const SaArgs &p, const SaSpace &sp, uint32_t block, uint8_t *vt) {
    const int lane = threadIdx.x & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wide = (uint32_t)(p.HK + SA_WAVES - 1) / SA_WAVES, q8 = block >> 3, grp = q8 / wide;
    const uint32_t piece = grp * 8 + (block & 7);  // the heads of a piece to one XCD
    const int h = (int)((q8 - grp * wide) * SA_WAVES) + wave;
    int v = 0;
    int blk0 = 0, per = 1;
    const SaLanes lanes = PRE ? sa_lanes(p) : SaLanes{};
    if (!sa_piece<PRE>(p, lanes, sp, piece, block == 0 && wave == 0, v, blk0, per)) return;
    if (h >= p.HK) return;
    const int64_t W = (int64_t)p.HK * CA_D, C = PRE ? p.CP : p.C;
    const SaTile tile = PRE ? sa_tile(p, lanes, v) : SaTile{v / p.ntile, 0, p.S * p.G, (v % p.ntile) * sp.rows};
    const int64_t len = PRE ? sa_prefix_length(p, tile.prefix) : sa_clamp(p.lengths[tile.prefix], p.C);
    const int requests = PRE ? sa_requests(p, lanes, tile.prefix) : 0;
    const int64_t base = (int64_t)tile.prefix * C * W + h * CA_D;
    const CaKeys keys{(PRE ? p.pk : p.kc) + base, (PRE ? p.pks : p.ks) + base / 32, (PRE ? p.pv : p.vc) + base,
                      (PRE ? p.pvs : p.vs) + base / 32, C, W, len};
    const int nblk = (int)((len + CA_KB - 1) / CA_KB), blk1 = blk0 + per < nblk ? blk0 + per : nblk;
    f32x4_t o[NR][8];
    float m[NR], l[NR];
    ca_wave<NR>(keys, blk0, blk1, p.scale_log2e, !PRE && p.tree ? len - p.S : len, vt,
                [&](int t, uint64_t &bits) {
                    int r = tile.row0 + 16 * t + lr;
                    r = r < tile.rows ? r : tile.rows - 1;  // rows past the end: computed, not stored
                    const int sg = p.S * p.G, i = PRE ? r / sg : 0, in = r - i * sg, s = in / p.G;
                    const int b = PRE ? sa_request(p, tile, requests, i) : tile.prefix;
                    bits = PRE ? 0 : ca_tree_bits(p.tree ? p.tree + b * p.tree_b + s * p.S : nullptr, p.S);
                    return p.q + b * p.ldqb + s * p.ldq + (h * p.G + (in - s * p.G)) * CA_D;
                },
                o, m, l);
#pragma unroll
    for (int t = 0; t < NR; ++t) {
        float lt = l[t] + __shfl_xor(l[t], 16, 64);
        lt += __shfl_xor(lt, 32, 64);
        if (tile.row0 + 16 * t + lr >= tile.rows) continue;
        const int64_t at = ((int64_t)piece * p.HK + h) * sp.rows + 16 * t + lr;
        float *dst = sp.part_o + at * CA_D + 4 * kg;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4_t *>(dst + 16 * dt) = o[t][dt];
        if (kg == 0) sp.part_ml[at] = make_float2(m[t], lt);
    }
}

template <int NP, int NO>
__global__ __launch_bounds__(64 * SA_WAVES, 2) void k_shared_attn(SaArgs p) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[SA_WAVES * CA_VTILE];
    uint8_t *const vt = lds + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * CA_VTILE;
    if (blockIdx.x < p.pre.blocks) sa_wave<true, NP>(p, p.pre, blockIdx.x, vt);
    else sa_wave<false, NO>(p, p.own, blockIdx.x - p.pre.blocks, vt);
}

// Many rows to a prefix: a workgroup of four waves takes 32 RG rows and blocks of 64 keys; a wave 32 rows and, of each
// block, all keys (RG 4) or one half of them (RG 2).  The block's codes become bf16 once, in LDS, where the wave above
// converts for 16 or 32 rows of its own.  RG 2, bound by memory: two buffers, two blocks on their way in registers, two
// workgroups a CU; waves of the same rows join in LDS.  RG 4, bound by the instructions that a wave issues one after
// the other: one buffer and one block on its way, so that three workgroups' registers fit a CU; a request's own keys
// go in tiles of 16 rows there, which fit too (with two of everything, us: 96 rows of 32 heads over 8392 keys 61 for
// 46; 128 of 8 heads over 32768 59 for 49; but 64-row tiles of one buffer 93 for 87 over five long prefixes).
// Rows of K are 16 bytes longer than a key, of V 32: a K operand's 16 rows, and the 8 rows that half a wave reads
// transposed, lie in different banks, and every read is one address and a constant.
constexpr int ST_KEYS = 64, ST_K = 2 * CA_D + 16, ST_V = 2 * CA_D + 32, ST_VAT = ST_KEYS * ST_K, ST_BUF = ST_VAT + ST_KEYS * ST_V;
template <int RG, int NO>
__global__ __launch_bounds__(64 * SA_WAVES, RG == 4 ? 3 : 2) void k_shared_tile(SaArgs p) {
    constexpr int KQ = 4 / RG, DEPTH = RG == 4 ? 1 : 2;                   // waves of the same rows; buffers
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];      // DEPTH * ST_BUF
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rg = wave % RG, kq = wave / RG;
    if (blockIdx.x >= p.pre.blocks) {
        sa_wave<false, NO>(p, p.own, blockIdx.x - p.pre.blocks, lds + wave * CA_VTILE);
        return;
    }
    // Eight heads of a piece to one XCD: they read neighbouring lines, and the same ones of exponents.
    const uint32_t q8 = blockIdx.x >> 3, unit = (q8 >> 3) * 8 + (blockIdx.x & 7), units = (uint32_t)(p.HK + 7) / 8;
    const uint32_t piece = unit / units;
    const int h = (int)(unit - piece * units) * 8 + (int)(q8 & 7);
    int v = 0;
    int blk0 = 0, per = 1;
    const SaLanes lanes = sa_lanes(p);
    if (!sa_piece<true>(p, lanes, p.pre, piece, blockIdx.x == 0 && wave == 0, v, blk0, per) || h >= p.HK) return;
    const SaTile tile = sa_tile(p, lanes, v);
    const int requests = sa_requests(p, lanes, tile.prefix);
    const int64_t len = sa_prefix_length(p, tile.prefix), W = (int64_t)p.HK * CA_D, base = (int64_t)tile.prefix * p.CP * W + h * CA_D;
    const int nblk = (int)((len + ST_KEYS - 1) / ST_KEYS), blk1 = blk0 + per < nblk ? blk0 + per : nblk;
    const float c = p.scale_log2e, ninf = -__builtin_inff();

    // A thread's share of a block: 16 codes of K and of V of keys tid / 8 and tid / 8 + 32.  Wave-uniform bases and
    // 32-bit offsets; only a block that reaches past the cache's end clamps its keys to the last.
    const int ck = tid >> 3, cc = tid & 7;
    struct Raw {
        uint4 k[2], v[2];
        uint32_t ke[2], ve[2];
    };
    const uint32_t w32 = (uint32_t)W;
    const uint8_t *const pk = p.pk + base, *const pv = p.pv + base, *const pks = p.pks + base / 32, *const pvs = p.pvs + base / 32;
    auto load = [&](Raw &w, int blk) {
        blk = blk < blk1 ? blk : blk1 - 1;  // (past the end: not converted)
        const int64_t k0 = (int64_t)blk * ST_KEYS, b8 = k0 * W, b5 = k0 * (W / 32);
        const int last = p.CP - k0 < ST_KEYS ? (int)(p.CP - k0) - 1 : ST_KEYS - 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t key = 32 * i + ck < last ? 32 * i + ck : last, at = key * w32 + 16 * cc, ae = key * (w32 / 32) + (cc >> 1);
            w.k[i] = *reinterpret_cast<const uint4 *>(pk + b8 + at);
            w.v[i] = *reinterpret_cast<const uint4 *>(pv + b8 + at);
            w.ke[i] = (pks + b5)[ae];
            w.ve[i] = (pvs + b5)[ae];
        }
    };
    bf16x8_t qf[2][4];  // d [64 j + 16 kg + 8 half, + 8) in step 2 j + half
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        int r = tile.row0 + 32 * rg + 16 * t + lr;
        r = r < tile.rows ? r : tile.rows - 1;
        const int sg = p.S * p.G, i = r / sg, in = r - i * sg, sq = in / p.G;
        const int b = sa_request(p, tile, requests, i);
        const uint16_t *qr = p.q + b * p.ldqb + sq * p.ldq + (h * p.G + (in - sq * p.G)) * CA_D + 16 * kg;
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[t][j] = *reinterpret_cast<const bf16x8_t *>(qr + 64 * (j >> 1) + 8 * (j & 1));
    }
    Raw raw[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) load(raw[i], blk0 + i);
    // Q is waited for here: a wait inside the loop would be one for all loads before the last, the second block's too.
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(qf[t][j]));
    f32x4_t o[2][8];
    float m[2], l[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        m[t] = ninf;
        l[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[t][dt] = f32x4_t{};
    }
    const bool idle = tile.row0 + 32 * rg >= tile.rows;  // no rows of this wave's: it only converts
    // Places of this lane's operands in a buffer: K's chunks of row lr, V's units of key 4 kg + lr / 4.
    const int vkey = 4 * kg + (lr >> 2);
    const uint8_t *const kat = lds + (32 * kq + lr) * ST_K + 32 * kg;
    const uint32_t vat = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds + ST_VAT + (32 * kq + vkey) * ST_V + (lr & 3) * 8;
    typedef __attribute__((address_space(3))) i16x4_t *tr_t;
    auto convert = [&](const Raw &w, int blk, int buf) {
        const int live = len - (int64_t)blk * ST_KEYS < ST_KEYS ? (int)(len - (int64_t)blk * ST_KEYS) : ST_KEYS;
        uint8_t *const kb = lds + buf * ST_BUF + ck * ST_K + 32 * cc, *const vb = lds + buf * ST_BUF + ST_VAT + ck * ST_V + 32 * cc;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int key = 32 * i + ck;
            const float ks = mx_scale_operand((int)w.ke[i]);
            *reinterpret_cast<bf16x8_t *>(kb + 32 * i * ST_K) = ca_operand(w.k[i].x, w.k[i].y, ks);
            *reinterpret_cast<bf16x8_t *>(kb + 32 * i * ST_K + 16) = ca_operand(w.k[i].z, w.k[i].w, ks);
            uint4 x = w.v[i];
            uint32_t e = w.ve[i];
            if (key >= live) {  // V past the last key is zeros, whatever the cache holds there
                x = make_uint4(0, 0, 0, 0);
                e = 0;
            }
            const float vs = mx_scale_operand((int)e);
            *reinterpret_cast<bf16x8_t *>(vb + 32 * i * ST_V) = ca_operand(x.x, x.y, vs);
            *reinterpret_cast<bf16x8_t *>(vb + 32 * i * ST_V + 16) = ca_operand(x.z, x.w, vs);
        }
    };
    // 32 keys of the block in a buffer, the wave's first or (RG 4) second 32, for its 32 rows; `left` keys are there.
    auto attend = [&](int buf, int half, int64_t left) {
        f32x4_t s[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bf16x8_t kf = *reinterpret_cast<const bf16x8_t *>(kat + (buf * ST_BUF + (32 * half + 16 * u) * ST_K + 128 * (j >> 1) + 16 * (j & 1)));
#pragma unroll
                for (int t = 0; t < 2; ++t) s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[t][j], j == 0 ? f32x4_t{} : s[t][u], 0, 0, 0);
            }
        u32x4_t pw[2], pl[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (left < 32) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][u][i] = 16 * u + 4 * kg + i < (int)left ? s[t][u][i] : ninf;
            }
            float mx = ca_max(ca_max(ca_max(s[t][0][0], s[t][0][1]), ca_max(s[t][0][2], s[t][0][3])),
                              ca_max(ca_max(s[t][1][0], s[t][1][1]), ca_max(s[t][1][2], s[t][1][3])));
            // m follows the row's maximum when a score has passed it by more than 2^8: till then p is at most 2^8, which
            // numerator and sum hold as well.
            mx *= c;
            if (__builtin_amdgcn_ballot_w64(!(mx <= m[t] + 8.0f))) {
                const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
                mx = ca_swap_max(ca_max(__uint_as_float(sw[0]), __uint_as_float(sw[1])));
                const float mn = mx <= m[t] + 8.0f ? m[t] : ca_max(m[t], mx);  // (this row's own need, whoever else asked)
                const float alpha = __builtin_amdgcn_exp2f(m[t] - (mn == ninf ? 0.f : mn));
                m[t] = mn;
                l[t] *= alpha;
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) o[t][dt] *= alpha;
            }
            const float ref = m[t] == ninf ? 0.f : m[t];
            float e[8], sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i >> 2][i & 3], c, -ref));
                sum += e[i];
            }
            l[t] += sum;
            // p as two bf16 terms, as in ca_wave.
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                pw[t][i] = pack_bf16x2(e[2 * i], e[2 * i + 1]);
                pl[t][i] = pack_bf16x2(e[2 * i] - bf_lo(pw[t][i]), e[2 * i + 1] - bf_hi(pw[t][i]));
            }
        }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            const uint32_t at = vat + (buf * ST_BUF + 32 * half * ST_V + 32 * dt);
            const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<tr_t>((uintptr_t)at));
            const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<tr_t>((uintptr_t)(at + 16 * ST_V)));
            const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8_t, pl[t]), o[t][dt], 0, 0, 0);
                o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8_t, pw[t]), o[t][dt], 0, 0, 0);
            }
        }
    };
    auto block = [&](Raw &w, int blk, int buf) {
        if (DEPTH == 1) __syncthreads();  // the block before has been read
        convert(w, blk, buf);
        if (DEPTH == 1) load(w, blk + 1);
        __syncthreads();
        if (DEPTH == 2) load(w, blk + 2);
        if (idle) return;
#pragma unroll
        for (int i = 0; i < 2 / KQ; ++i) {
            const int64_t left = len - ((int64_t)blk * ST_KEYS + 32 * (kq + i));
            if (left > 0) attend(buf, i, left);
        }
    };
    for (int blk = blk0; blk < blk1; blk += DEPTH) {
        block(raw[0], blk, 0);
        if (DEPTH == 2 && blk + 1 < blk1) block(raw[DEPTH - 1], blk + 1, 1);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        l[t] += __shfl_xor(l[t], 16, 64);
        l[t] += __shfl_xor(l[t], 32, 64);
    }
    // The second wave of the same rows joins with the first.
    if constexpr (KQ == 2) {
        f32x4_t *const so = reinterpret_cast<f32x4_t *>(lds) + rg * (16 * 64);
        float2 *const sml = reinterpret_cast<float2 *>(lds + RG * (32 * CA_D * 4)) + rg * 32;
        __syncthreads();
        if (kq) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) so[(t * 8 + dt) * 64 + lane] = o[t][dt];
                if (kg == 0) sml[t * 16 + lr] = make_float2(m[t], l[t]);
            }
        }
        __syncthreads();
        if (kq) return;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const float2 other = sml[t * 16 + lr];
            const float M = ca_max(m[t], other.x), ref = M == ninf ? 0.f : M;
            const float w0 = __builtin_amdgcn_exp2f(m[t] - ref), w1 = __builtin_amdgcn_exp2f(other.x - ref);
            m[t] = M;
            l[t] = l[t] * w0 + other.y * w1;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) o[t][dt] = o[t][dt] * w0 + so[(t * 8 + dt) * 64 + lane] * w1;
        }
    }
    if (idle) return;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int r = 32 * rg + 16 * t + lr;
        if (tile.row0 + r >= tile.rows) continue;
        const int64_t at = ((int64_t)piece * p.HK + h) * p.pre.rows + r;
        float *dst = p.pre.part_o + at * CA_D + 4 * kg;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4_t *>(dst + 16 * dt) = o[t][dt];
        if (kg == 0) p.pre.part_ml[at] = make_float2(m[t], l[t]);
    }
}

template <int RG, int NO>
static int launch_shared_tile(const SaArgs &a, dim3 grid, hipStream_t st) {
    constexpr int bytes = (RG == 4 ? 1 : 2) * ST_BUF;
    static std::atomic<bool> done[QIM_MAX_DEVICES];
    if (bytes > 65536) {
        const int rc = reserve_lds(reinterpret_cast<const void *>(k_shared_tile<RG, NO>), bytes, done, "qim_attention_shared");
        if (rc != QIM_OK) return rc;
    }
    launch(k_shared_tile<RG, NO>, grid, dim3(64 * SA_WAVES), bytes, st, a);
    return QIM_OK;
}

// Join the pieces of a row: GP groups of 32 lanes (4 head dims each) take them in turn, four loads at a time, and join in
// LDS.  A row's pieces are its prefix's, then its own.
template <int GP>
__global__ __launch_bounds__(256) void k_shared_join(SaArgs p, int64_t nrows) {
    __shared__ float4 so[8][32];
    __shared__ float2 sml[8];
    const int grp = threadIdx.x >> 5, ln = threadIdx.x & 31;
    const int64_t g = (int64_t)blockIdx.x * (8 / GP) + grp / GP;
    const bool live = g < nrows;
    const int sg = p.S * p.G;
    const int64_t row = live ? g : 0, item = row / sg;
    const int r = (int)(row - item * sg), b = (int)(item / p.HK), h = (int)(item - (int64_t)b * p.HK);
    const int2 od = p.own.dir[b * p.ntile + r / p.own.rows];
    int2 w = make_int2(0, b);
    if (p.few) {
        const int mine = (threadIdx.x & 63) < p.B ? p.share[threadIdx.x & 63] : -1, prefix = p.share[b];
        w.x = -1;
        sa_each_prefix(p, mine, [&](int i, uint64_t all, int first, int) {
            if (prefix == i) w = make_int2(first, (int)__builtin_popcountll(all & ((1ull << b) - 1)));
        });
    } else if (p.share) {
        w = p.where[b];
    }
    int2 pd = make_int2(0, 0);
    int pr = 0;
    if (w.x >= 0) {
        const int64_t rr = (int64_t)w.y * sg + r;
        pd = p.pre.dir[w.x + (int)(rr / p.pre.rows)];
        pr = (int)(rr % p.pre.rows);
    }
    const int64_t pstep = (int64_t)p.HK * p.pre.rows, ostep = (int64_t)p.HK * p.own.rows;
    const int64_t pfirst = pd.x * pstep + (int64_t)h * p.pre.rows + pr, ofirst = od.x * ostep + (int64_t)h * p.own.rows + r % p.own.rows;
    const int n = pd.y + od.y;
    const float ninf = -__builtin_inff();
    float M = ninf, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = grp % GP; i < n; i += 4 * GP) {
        float2 ml[4];
        float4 f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = i + j * GP < n ? i + j * GP : i;
            const bool pre = c < pd.y;
            const int64_t at = pre ? pfirst + c * pstep : ofirst + (c - pd.y) * ostep;
            ml[j] = (pre ? p.pre : p.own).part_ml[at];
            f[j] = *reinterpret_cast<const float4 *>((pre ? p.pre : p.own).part_o + at * CA_D + 4 * ln);
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
            const float e = __builtin_amdgcn_exp2f(ml[j].x - ref);
            if (i + j * GP < n) {  // (a repeated piece may hold NaN)
                L += ml[j].y * e;
                acc = make_float4(acc.x + f[j].x * e, acc.y + f[j].y * e, acc.z + f[j].z * e, acc.w + f[j].w * e);
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
            const float e = __builtin_amdgcn_exp2f(sml[grp + j].x - ref);
            const float4 f = so[grp + j][ln];
            L += sml[grp + j].y * e;
            acc = make_float4(acc.x + f.x * e, acc.y + f.y * e, acc.z + f.z * e, acc.w + f.w * e);
        }
    }
    if (!live) return;
    const float inv = L == 0.f ? 0.f : 1.0f / L;  // no visible key: zeros
    const int s = r / p.G, head = h * p.G + (r - s * p.G);
    uint16_t *dst = p.o + (((int64_t)b * p.S + s) * p.H + head) * CA_D + 4 * ln;
    *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

// Row tiles and the pieces' numbers.
struct SaPlan {
    int64_t rg, np, no, ntile, tr, keys;  // rg: row groups of a tile (0: tiles of 16 np rows, a wave each); tr: rows of a prefix tile
    int64_t vp, vo, gp, go;               // sequences, pieces (at most)
    int64_t wp, wo;                       // workgroups of a piece's heads
    int64_t HK, B;
    bool shared, few;
    static int64_t up(int64_t n) { return (n + 255) / 256 * 256; }
    int64_t blocks_p() const { return rg ? (gp * ((HK + 7) / 8) + 7) / 8 * 64 : (gp + 7) / 8 * 8 * wp; }
    int64_t blocks_o() const { return (go + 7) / 8 * 8 * wo; }
    int64_t rows_p() const { return gp * HK * tr; }
    int64_t rows_o() const { return go * HK * no * 16; }
    int64_t bytes() const {
        return up(rows_p() * CA_D * 4) + up(rows_o() * CA_D * 4) + up(rows_p() * 8) + up(rows_o() * 8) + up(vp * 8) + up(vo * 8) +
               (shared && !few ? up(vp * 16) + up(B * 4) + up(B * 8) : 0);
    }
};
static SaPlan sa_plan(int64_t B, int64_t S, int64_t CP, int64_t C, int64_t H, int64_t HK, int64_t P, bool shared) {
    SaPlan pl;
    const int64_t sg = S * (H / HK), rows = B * sg, cus = device_cus() > 0 ? device_cus() : 256;
    const int64_t each = ((B + P - 1) / P) * sg;  // rows of a prefix, if they are alike
    pl.HK = HK;
    pl.B = B;
    pl.shared = shared;
    pl.rg = each <= 32 ? 0 : each <= 64 ? 2 : 4;
    pl.np = each > 16 ? 2 : 1;
    pl.tr = pl.rg ? 32 * pl.rg : 16 * pl.np;
    pl.keys = pl.rg ? ST_KEYS : CA_KB;
    pl.no = sg > 16 && pl.rg != 4 ? 2 : 1;
    pl.wo = (HK + SA_WAVES - 1) / SA_WAVES;
    pl.wp = pl.rg ? HK : pl.wo;
    pl.ntile = (sg + 16 * pl.no - 1) / (16 * pl.no);
    pl.vo = B * pl.ntile;
    // Several prefixes: each may end with a tile that is not full.
    pl.vp = (rows + pl.tr - 1) / pl.tr + (shared && P > 1 ? (P - 1 < B ? P - 1 : B) : 0);
    pl.few = shared && B <= 64 && P <= SA_FEW_PREFIXES && pl.vp <= 64;
    const int64_t bp = (CP + pl.keys - 1) / pl.keys, bo = (C + CA_KB - 1) / CA_KB;
    // The pieces of both spaces together: two workgroups a CU, divided by the time that the spaces' blocks take one
    // (measured: 1.0 and 1.5 us for a wave's 16 and 32 rows, 1.4 and 2.3 us for tiles of 64 and 128).  Three of a CU's
    // workgroups of 128 rows run at once; a third pays where a piece stays long beside its start and its results (8392 keys,
    // requests of 24 rows on 32 heads, two and three a CU: 6 requests 73.8 and 68.8 us, 12 104 and 95.5; 4, pieces of 6 blocks,
    // 46.4 and 48.9; 32 of 4 rows on 8 heads over 32768 keys 49.4 and 51.1).
    const double wave[2] = {1.0, 1.5};
    const double tp = (double)bp * pl.vp * pl.wp * (pl.rg == 4 ? 2.3 : pl.rg == 2 ? 1.4 : wave[pl.np - 1]), to = (double)bo * pl.vo * pl.wo * wave[pl.no - 1];
    int64_t wgs = pl.rg == 4 ? 3 : 2;
    // At least a piece a sequence (also where a space holds no keys: its first workgroup writes dir), at most one a block.
    auto pieces = [&](double w, int64_t v, int64_t blocks, int64_t wide) {
        int64_t n = (int64_t)(wgs * cus * w / (tp + to) / wide + 0.5);
        const int64_t most = v * blocks;
        if (n < 4 * v) n = n / v * v;  // (whole pieces of sequences that are alike)
        return n < v || most < v ? v : n < most ? n : most;
    };
    if (pl.rg == 4 && bp * pl.vp < 10 * pieces(tp, pl.vp, bp, pl.wp)) wgs = 2;
    pl.gp = pieces(tp, pl.vp, bp, pl.wp);
    pl.go = pieces(to, pl.vo, bo, pl.wo);
    return pl;
}

}  // namespace qim

using namespace qim;

static bool sa_shape(int64_t B, int64_t S, int64_t CP, int64_t C, int64_t H, int64_t HK, int64_t P, int shared) {
    if (!(B > 0 && S > 0 && S <= CA_MAX_S && P > 0 && P <= SA_MAX_PREFIXES && (shared || P == 1) && CP > 0 && C >= 0 && CP < (1ll << 31) &&
          C < (1ll << 31) && HK > 0 && H > 0 && H % HK == 0 && H <= (1 << 16) && B < (1 << 20) && B * S * (H / HK) < (1 << 24) &&
          B * C < (1ll << 40) / HK && P * CP < (1ll << 40) / HK))
        return false;
    const SaPlan pl = sa_plan(B, S, CP, C, H, HK, P, shared);
    return (pl.blocks_p() + pl.blocks_o()) * (64 * SA_WAVES) < (1ll << 32) && B * S * H < (1ll << 26) && pl.vp * ((CP + 31) / 32) < (1ll << 31) &&
           pl.vo * ((C + 31) / 32) < (1ll << 31);
}

extern "C" int64_t qim_attention_shared_workspace_bytes(int64_t B, int64_t S, int64_t CP, int64_t C, int64_t H, int64_t HK, int64_t P,
                                                        int shared) {
    return sa_shape(B, S, CP, C, H, HK, P, shared) ? sa_plan(B, S, CP, C, H, HK, P, shared).bytes() : 0;
}

extern "C" int qim_attention_shared(const void *q, int64_t ldqb, int64_t ldq, const void *pk, const void *pks, const void *pv,
                                    const void *pvs, const int32_t *prefix_lengths, const int32_t *share, const void *kc,
                                    const void *ks, const void *vc, const void *vs, const int32_t *lengths, const void *tree,
                                    int64_t tree_b, void *o, void *workspace, int64_t workspace_bytes, int64_t B, int64_t S,
                                    int64_t P, int64_t CP, int64_t C, int64_t H, int64_t HK, int64_t D, float scale, void *stream) {
    const char *who = "qim_attention_shared";
    QIM_REQUIRE(q && pk && pks && pv && pvs && kc && ks && vc && vs && lengths && o && workspace, QIM_ERR_ARG, "%s: null pointer", who);
    QIM_REQUIRE(D == CA_D, QIM_ERR_SHAPE, "%s: head dim %lld (128 only)", who, (long long)D);
    QIM_REQUIRE(scale > 0.0f && scale < 1e30f, QIM_ERR_ARG, "%s: scale must be positive and finite", who);
    QIM_REQUIRE(sa_shape(B, S, CP, C, H, HK, P, share ? 1 : 0), QIM_ERR_SHAPE,
                "%s: B %lld, S %lld (1..64), %lld prefixes of %lld (one without share), C %lld, %lld heads on %lld K/V heads", who,
                (long long)B, (long long)S, (long long)P, (long long)CP, (long long)C, (long long)H, (long long)HK);
    QIM_REQUIRE(ldq >= H * D && ldqb >= 0 && ldq % 8 == 0 && ldqb % 8 == 0 && tree_b >= 0 && aligned16(q) && aligned16(pk) &&
                    aligned16(pks) && aligned16(pv) && aligned16(pvs) && aligned16(kc) && aligned16(ks) && aligned16(vc) && aligned16(vs) &&
                    aligned16(o) && aligned16(workspace) && ((reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(prefix_lengths) |
                    reinterpret_cast<uintptr_t>(share)) & 3u) == 0,
                QIM_ERR_LAYOUT, "%s: rows and the workspace must be 16-byte aligned", who);
    const SaPlan pl = sa_plan(B, S, CP, C, H, HK, P, share != nullptr);
    QIM_REQUIRE(workspace_bytes >= pl.bytes(), QIM_ERR_ARG, "%s: workspace of %lld bytes, this problem needs %lld", who,
                (long long)workspace_bytes, (long long)pl.bytes());
    // Rows are written while others are still read, and the last launch reads lengths and workspace.
    const struct {
        const void *at;
        int64_t bytes;
    } inputs[] = {{q, 2 * ((B - 1) * ldqb + (S - 1) * ldq + H * D)}, {pk, P * CP * HK * D}, {pks, P * CP * HK * D / 32}, {pv, P * CP * HK * D},
                  {pvs, P * CP * HK * D / 32}, {kc, B * C * HK * D}, {ks, B * C * HK * D / 32}, {vc, B * C * HK * D}, {vs, B * C * HK * D / 32},
                  {prefix_lengths, 4 * P}, {share, 4 * B}, {lengths, 4 * B}, {tree, (B - 1) * tree_b + S * S}};
    for (const auto &in : inputs)
        QIM_REQUIRE(!in.at || !in.bytes || (!bytes_share(o, 2 * B * S * H * D, in.at, in.bytes) && !bytes_share(workspace, pl.bytes(), in.at, in.bytes)),
                    QIM_ERR_ARG, "%s: o or the workspace overlaps an input", who);
    QIM_REQUIRE(!bytes_share(o, 2 * B * S * H * D, workspace, pl.bytes()), QIM_ERR_ARG, "%s: o overlaps the workspace", who);
    uint8_t *at = static_cast<uint8_t *>(workspace);
    auto take = [&](int64_t n) {
        uint8_t *r = at;
        at += SaPlan::up(n);
        return r;
    };
    SaArgs a{};
    a.q = (const uint16_t *)q;
    a.ldqb = ldqb;
    a.ldq = ldq;
    a.pk = (const uint8_t *)pk, a.pks = (const uint8_t *)pks, a.pv = (const uint8_t *)pv, a.pvs = (const uint8_t *)pvs;
    a.kc = (const uint8_t *)kc, a.ks = (const uint8_t *)ks, a.vc = (const uint8_t *)vc, a.vs = (const uint8_t *)vs;
    a.lengths = lengths, a.plengths = prefix_lengths, a.share = share;
    a.tree = (const uint8_t *)tree;
    a.tree_b = tree_b, a.CP = CP, a.C = C;
    a.o = (uint16_t *)o;
    a.pre.part_o = (float *)take(pl.rows_p() * CA_D * 4);
    a.own.part_o = (float *)take(pl.rows_o() * CA_D * 4);
    a.pre.part_ml = (float2 *)take(pl.rows_p() * 8);
    a.own.part_ml = (float2 *)take(pl.rows_o() * 8);
    a.pre.dir = (int2 *)take(pl.vp * 8);
    a.own.dir = (int2 *)take(pl.vo * 8);
    a.few = pl.few;
    if (share && !pl.few) {
        a.tiles = (int4 *)take(pl.vp * 16);
        a.order = (int32_t *)take(B * 4);
        a.where = (int2 *)take(B * 8);
    }
    a.pre.V = (int)pl.vp, a.pre.most = (int)pl.gp, a.pre.rows = (int)pl.tr, a.pre.keys = (int)pl.keys, a.pre.blocks = (uint32_t)pl.blocks_p();
    a.own.V = (int)pl.vo, a.own.most = (int)pl.go, a.own.rows = (int)(16 * pl.no), a.own.keys = CA_KB, a.own.blocks = (uint32_t)pl.blocks_o();
    a.B = (int)B, a.S = (int)S, a.H = (int)H, a.HK = (int)HK, a.G = (int)(H / HK), a.P = (int)P, a.ntile = (int)pl.ntile;
    a.scale_log2e = scale * 1.4426950408889634f;
    hipStream_t st = as_stream(stream);
    if (share && !pl.few) launch(k_shared_plan, dim3(1), dim3(1024), (size_t)(8 * P), st, a);
    const dim3 grid(a.pre.blocks + a.own.blocks);
    if (pl.rg) {
        const int rc = pl.rg == 4 ? launch_shared_tile<4, 1>(a, grid, st) : pl.no == 2 ? launch_shared_tile<2, 2>(a, grid, st) : launch_shared_tile<2, 1>(a, grid, st);
        if (rc != QIM_OK) return rc;
    } else {
        launch(pl.np == 2 ? (pl.no == 2 ? k_shared_attn<2, 2> : k_shared_attn<2, 1>) : (pl.no == 2 ? k_shared_attn<1, 2> : k_shared_attn<1, 1>),
               grid, dim3(64 * SA_WAVES), 0, st, a);
    }
    const int64_t nrows = B * HK * S * a.G, each = pl.gp / pl.vp + pl.go / pl.vo;
    const int64_t gp = each > 16 ? 8 : each > 4 ? 2 : 1;
    launch(gp == 8 ? k_shared_join<8> : gp == 2 ? k_shared_join<2> : k_shared_join<1>, dim3((unsigned)((nrows * gp + 7) / 8)), dim3(256), 0, st,
           a, nrows);
    return check_launch(who);
}
