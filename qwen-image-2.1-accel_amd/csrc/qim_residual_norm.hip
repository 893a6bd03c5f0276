// The gated residual of a block with the norms on both of its sides, one pass over the rows:
//
//   u = post(x),  h' = h + alpha * gate * u,  z = norm(h') * scale + shift
//
// post: none, RMSNorm (times its weight) or LayerNorm without affine; norm: one of the two.
// gate, scale, shift: a vector per sequence or one for all.  h' leaves in bf16, z in bf16 or as the
// MXFP8 codes and exponents of the GEMM's input.
//
// Two forms.  Rounded once: everything in fp32 with the row sums in float64, h' and z rounded at their
// ends, z taken from the unrounded h'.  Eager (post none, LayerNorm, alpha 1): every step rounded to
// bf16 as qim_gated_residual followed by qim_adaln / qim_adaln_quantize round it, the same bits.
//
// Memory-bound: 8 bytes an element (7.03 with MXFP8) for about 20 vector operations.  A workgroup takes a
// row; its lanes hold their 16-byte vectors of the row in registers from the loads to the stores, so the
// reductions between (one for post, one for norm) cost no second read.  Measured at D 4096: 2048 rows with gate, scale and
// shift 14 us, 4.8 TB/s; 16384 rows with a norm on both sides 109-112 us, 4.8-4.9 TB/s, of the 5.1 that a 1 GiB copy reaches;
// 16 rows 4.1 us, a launch and two reductions.  The eager form beside the two launches that it replaces (D 4096, from a graph, bf16
// and MXFP8): 16 rows 3.3 us for 5.2 and 3.7 for 6.0; 2048 17.1 for 18.6 and 16.8 for 18.9; 16384 98 for 109 and 99 for 108.
#include "qim_device.h"
#include "qim_runtime.h"

namespace qim {

struct ResNormArgs {
    const uint16_t *h, *x, *post_w, *gate, *norm_w, *scale, *shift;
    uint16_t *ho, *z;
    uint8_t *q, *qs;
    int64_t ldh, ldx, ldho, ldz, gate_b, scale_b, shift_b;
    int64_t rows, rows_pad;
    int D, post, norm, add_one, tiled;
    uint32_t seq;
    float alpha, post_eps, norm_eps;
    double inv_d;
};

constexpr int RN_MAX_WAVES = 16;

// Sums of two values over the workgroup, in one fixed order.  `slot` alternates between calls, so that one
// barrier a call is enough.
template <bool TWO>
__device__ __forceinline__ void rn_sum(double &a, double &b, double (*red)[2][RN_MAX_WAVES], int slot) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
    a = wave_total(a);
    if (TWO) b = wave_total(b);
    if (nw == 1) return;
    if (lane == 0) {
        red[slot][0][wave] = a;
        if (TWO) red[slot][1][wave] = b;
    }
    __syncthreads();
    a = b = 0.0;
    for (int w = 0; w < nw; ++w) {
        a += red[slot][0][w];
        if (TWO) b += red[slot][1][w];
    }
}

// Mean (as an fp32 pair) and reciprocal deviation of a row from its float64 sums.  The difference s2/D - mean^2 of
// float64 sums keeps 2^-53 of the mean's square; it is not below 0 by more than that.  A variance that
// fp32 does not hold (values around 1e19 and more) takes the float64 expression.
struct RnStat {
    float mean, mean_lo, rstd;
};
__device__ __forceinline__ RnStat rn_stat(int kind, double s1, double s2, double inv_d, float eps) {
    RnStat r;
    const double mean = kind == QIM_NORM_LAYER ? s1 * inv_d : 0.0;
    double var = s2 * inv_d - mean * mean;
    var = var < 0.0 ? 0.0 : var;
    r.mean = (float)mean;
    r.mean_lo = (float)(mean - (double)r.mean);
    r.rstd = var < 1e38 ? rstd_of((float)var, eps) : (float)(1.0 / sqrt(var + (double)eps));
    return r;
}

// z of one 16-byte vector to its place: bf16, or the codes (8 bytes) and the row's exponents (16 adjacent
// lanes own one dword of the swizzled array).
__device__ __forceinline__ void rn_store_codes(const ResNormArgs &p, int64_t row, int j, const uint2 &c, int e) {
    const int64_t at = p.tiled ? mxt_offset(row, (int64_t)j * 8, p.rows_pad, p.D) : row * p.D + (int64_t)j * 8;
    st_nt(p.q + at, c);
    const uint32_t e1 = dpp_mov<DPP_ROW_SHL4>((uint32_t)e), e2 = dpp_mov<DPP_ROW_SHL8>((uint32_t)e);
    const uint32_t e3 = dpp_mov<DPP_ROW_SHL12>((uint32_t)e);
    if ((threadIdx.x & 15) == 0)
        *reinterpret_cast<uint32_t *>(p.qs + mx_scale_offset(row, j >> 2, p.D)) = (uint32_t)e | (e1 << 8) | (e2 << 16) | (e3 << 24);
}

// NV 16-byte vectors a lane; lane t holds the vectors t, t + blockDim, ...
template <int NV, bool QUANT, bool EAGER>
__global__ __launch_bounds__(NV > 2 ? 256 : 64 * RN_MAX_WAVES) void k_residual_norm(ResNormArgs p) {
    __shared__ double red[2][2][RN_MAX_WAVES];
    const int tid = threadIdx.x, nthr = blockDim.x, nvec = p.D >> 3;
    const int64_t row = blockIdx.x;
    if (QUANT && row >= p.rows) {  // padding rows of the quantized output: codes 0, exponents 0
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (tid + nthr * i < nvec) rn_store_codes(p, row, tid + nthr * i, make_uint2(0, 0), 0);
        return;
    }
    const uint32_t b = (uint32_t)row / p.seq;
    const uint4 *hr = reinterpret_cast<const uint4 *>(p.h + row * p.ldh), *xr = reinterpret_cast<const uint4 *>(p.x + row * p.ldx);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4 xv[NV], hv[NV], gv[NV], pw[NV];
    auto rows_of = [&](const uint16_t *base, int64_t stride) { return reinterpret_cast<const uint4 *>(base + b * stride); };
    auto load = [&](uint4 (&v)[NV], const uint4 *from, bool stream) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = tid + nthr * i;
            v[i] = j < nvec ? (stream ? ld_nt(from + j) : from[j]) : zero;
        }
    };
    load(xv, xr, true);
    load(hv, hr, true);
    if (p.gate) load(gv, rows_of(p.gate, p.gate_b), false);
    if (!EAGER && p.post_w) load(pw, reinterpret_cast<const uint4 *>(p.post_w), false);

    float y[NV][8];  // x, then h'
#pragma unroll
    for (int i = 0; i < NV; ++i) unpack8(xv[i], y[i]);
    if constexpr (!EAGER) {
        if (p.post) {
            double s1 = 0.0, s2 = 0.0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    const double v = (double)y[i][t];
                    s1 += v;
                    s2 = __builtin_fma(v, v, s2);
                }
            rn_sum<true>(s1, s2, red, 0);
            const RnStat st = rn_stat(p.post, s1, s2, p.inv_d, p.post_eps);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int t = 0; t < 8; ++t) y[i][t] = ((y[i][t] - st.mean) - st.mean_lo) * st.rstd;
            if (p.post_w) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    float w[8];
                    unpack8(pw[i], w);
#pragma unroll
                    for (int t = 0; t < 8; ++t) y[i][t] *= w[t];
                }
            }
        }
    }
    if (p.gate) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float g[8];
            unpack8(gv[i], g);
#pragma unroll
            for (int t = 0; t < 8; ++t) y[i][t] = EAGER ? rbf(g[t] * y[i][t]) : y[i][t] * g[t];
        }
    }
    uint4 *ho = reinterpret_cast<uint4 *>(p.ho + row * p.ldho);
    double s1 = 0.0, s2 = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float h[8];
        unpack8(hv[i], h);
        const int j = tid + nthr * i;
#pragma unroll
        for (int t = 0; t < 8; ++t) y[i][t] = EAGER ? rbf(h[t] + y[i][t]) : __builtin_fmaf(p.alpha, y[i][t], h[t]);
        if (j >= nvec) {  // (a LayerNorm of x leaves -mean * rstd in absent vectors)
#pragma unroll
            for (int t = 0; t < 8; ++t) y[i][t] = 0.f;
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const double v = (double)y[i][t];
            s1 += v;
            s2 = __builtin_fma(v, v, s2);
        }
    }
    // The vectors of the second norm are on their way during its reduction.
    uint4 nw[NV], sv[NV], tv[NV];
    if (!EAGER && p.norm_w) load(nw, reinterpret_cast<const uint4 *>(p.norm_w), false);
    if (p.scale) load(sv, rows_of(p.scale, p.scale_b), false);
    if (p.shift) load(tv, rows_of(p.shift, p.shift_b), false);
    rn_sum<true>(s1, s2, red, 1);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = tid + nthr * i;
        if (j < nvec) st_nt(ho + j, pack8(y[i]));
    }
    float mean, mean_lo = 0.f, rstd;
    if constexpr (EAGER) {
        const double mean_d = s1 / (double)p.D;
        float var;
        if (!ln_variance(s2, mean_d, p.D, p.inv_d, var)) {  // uniform over the workgroup
            double ss = 0.0, none = 0.0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    const double d = tid + nthr * i < nvec ? (double)y[i][t] - mean_d : 0.0;
                    ss += d * d;
                }
            rn_sum<false>(ss, none, red, 0);
            var = (float)(ss / (double)p.D);
        }
        mean = (float)mean_d;
        rstd = rstd_of(var, p.norm_eps);
    } else {
        const RnStat st = rn_stat(p.norm, s1, s2, p.inv_d, p.norm_eps);
        mean = st.mean;
        mean_lo = st.mean_lo;
        rstd = st.rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = tid + nthr * i;
        if (j >= nvec) break;
        float *v = y[i], f[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] = EAGER ? rbf((v[t] - mean) * rstd) : ((v[t] - mean) - mean_lo) * rstd;
        if (!EAGER && p.norm_w) {
            unpack8(nw[i], f);
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] *= f[t];
        }
        if (p.scale) {
            unpack8(sv[i], f);
            if (p.add_one) {
#pragma unroll
                for (int t = 0; t < 8; ++t) f[t] = EAGER ? rbf(f[t] + 1.f) : f[t] + 1.f;
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] = EAGER ? rbf(v[t] * f[t]) : v[t] * f[t];
        }
        if (p.shift) {
            unpack8(tv[i], f);
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] += f[t];
        }
        if constexpr (!QUANT) {
            st_nt(reinterpret_cast<uint4 *>(p.z + row * p.ldz) + j, pack8(v));
        } else {
            int e;
            const uint2 c = EAGER ? quantize8_bf16(pack8(v), e) : quantize8(v, e);
            rn_store_codes(p, row, j, c, e);
        }
    }
}

template <bool QUANT, bool EAGER>
static void launch_residual_norm(const ResNormArgs &a, hipStream_t st) {
    const int nvec = a.D / 8;
    const dim3 grid((unsigned)a.rows_pad);
    auto go = [&](auto fn, int nv) { launch(fn, grid, dim3(64 * ((nvec + 64 * nv - 1) / (64 * nv))), 0, st, a); };
    // The eager form needs some 72 registers a lane: a row of more than 8 waves leaves a CU one or two workgroups, which wait at
    // their barriers with nothing beside them.  From 4096 to 8192 values it takes four vectors a lane instead, and no more than four
    // waves (4096 rows, us, the two separate calls, a vector a lane and four, bf16: D 4608 35.3, 38.2 and 30.4; 6144 44.6, 43.1 and
    // 37.8; 8192 58.7, 68.1 and 48.3; MXFP8: 37.2, 37.9 and 32.3; 46.5, 44.9 and 40.6; 58.9, 67.5 and 51.5).
    if constexpr (EAGER) {
        if (nvec > 512 && nvec <= 1024) {
            go(k_residual_norm<4, QUANT, EAGER>, 4);
            return;
        }
    }
    if (nvec <= 64 * RN_MAX_WAVES) go(k_residual_norm<1, QUANT, EAGER>, 1);
    else go(k_residual_norm<2, QUANT, EAGER>, 2);
}

}  // namespace qim

using namespace qim;

extern "C" int qim_residual_norm(const void *h, int64_t ldh, const void *x, int64_t ldx, int post, const void *post_weight,
                                 float post_eps, const void *gate, int64_t gate_b, float alpha, int norm,
                                 const void *norm_weight, float norm_eps, const void *scale, int64_t scale_b,
                                 const void *shift, int64_t shift_b, int flags, void *h_out, int64_t ldho, void *z,
                                 int64_t ldz, void *z_scales, int64_t M, int64_t D, int64_t seq, void *stream) {
    const char *who = "qim_residual_norm";
    QIM_REQUIRE(h && x && h_out && z, QIM_ERR_ARG, "%s: null pointer", who);
    QIM_REQUIRE(post >= QIM_NORM_NONE && post <= QIM_NORM_LAYER && (norm == QIM_NORM_RMS || norm == QIM_NORM_LAYER), QIM_ERR_ARG,
                "%s: post %d, norm %d", who, post, norm);
    QIM_REQUIRE((flags & ~(QIM_ADALN_ADD_ONE | QIM_ADALN_TILED | QIM_NORM_EAGER)) == 0, QIM_ERR_ARG, "%s: flags %d", who, flags);
    QIM_REQUIRE(!post_weight || post == QIM_NORM_RMS, QIM_ERR_ARG, "%s: a weight of no RMSNorm before the residual", who);
    QIM_REQUIRE(!norm_weight || norm == QIM_NORM_RMS, QIM_ERR_ARG, "%s: a weight of no RMSNorm after the residual", who);
    QIM_REQUIRE(scale || !(flags & QIM_ADALN_ADD_ONE), QIM_ERR_ARG, "%s: add_one without a scale", who);
    const bool eager = flags & QIM_NORM_EAGER;
    QIM_REQUIRE(!eager || (post == QIM_NORM_NONE && norm == QIM_NORM_LAYER && alpha == 1.0f && gate && scale), QIM_ERR_ARG,
                "%s: the eager form is the gated residual and LayerNorm * scale (+ shift)", who);
    QIM_REQUIRE(alpha - alpha == 0.0f, QIM_ERR_ARG, "%s: alpha is not finite", who);
    QIM_REQUIRE(!post || post_eps >= 0.0f, QIM_ERR_ARG, "%s: post_eps", who);
    QIM_REQUIRE(norm_eps >= 0.0f, QIM_ERR_ARG, "%s: norm_eps", who);
    QIM_REQUIRE(M > 0 && seq > 0 && D >= 8 && D % 8 == 0 && D <= 16384 && (!z_scales || D % 128 == 0), QIM_ERR_SHAPE,
                "%s: M %lld, seq %lld, D %lld (multiples of 8 up to 16384; of 128 for MXFP8)", who, (long long)M, (long long)seq, (long long)D);
    const int64_t pad = z_scales ? (M + 127) / 128 * 128 : M;
    QIM_REQUIRE(pad < (1ll << 22) && seq < (1ll << 31), QIM_ERR_SHAPE, "%s: too large", who);
    QIM_REQUIRE(ldh >= D && ldx >= D && ldho >= D && (z_scales || ldz >= D) && ldh % 8 == 0 && ldx % 8 == 0 && ldho % 8 == 0 &&
                    ldz % 8 == 0 && gate_b % 8 == 0 && scale_b % 8 == 0 && shift_b % 8 == 0 && gate_b >= 0 && scale_b >= 0 && shift_b >= 0,
                QIM_ERR_LAYOUT, "%s: rows must be multiples of 8 elements apart", who);
    QIM_REQUIRE(aligned16(h) && aligned16(x) && aligned16(h_out) && aligned16(z) && aligned16(z_scales) && aligned16(post_weight) &&
                    aligned16(norm_weight) && aligned16(gate) && aligned16(scale) && aligned16(shift),
                QIM_ERR_LAYOUT, "%s: operands must be 16-byte aligned", who);
    // A lane writes only where it has read: an output may be an input, row for row, and is else apart.
    auto apart = [&](const void *out, int64_t ldo, const void *t, int64_t ldt) {
        return (out == t && (ldo == ldt || M == 1)) || !rows_share(out, ldo, D, t, ldt, D, M);
    };
    bool ok = apart(h_out, ldho, h, ldh) && apart(h_out, ldho, x, ldx);
    if (z_scales) {
        const int64_t in[3] = {ldh, ldx, ldho};
        const void *rows[3] = {h, x, h_out};
        for (int i = 0; i < 3; ++i)
            ok = ok && !bytes_share(z, pad * D, rows[i], 2 * ((M - 1) * in[i] + D)) &&
                 !bytes_share(z_scales, pad * D / 32, rows[i], 2 * ((M - 1) * in[i] + D));
    } else {
        ok = ok && apart(z, ldz, h, ldh) && apart(z, ldz, x, ldx) && !rows_share(z, ldz, D, h_out, ldho, D, M);
    }
    // Other workgroups still read the vectors.
    const void *vectors[5] = {gate, scale, shift, post_weight, norm_weight};
    const int64_t steps[5] = {gate_b, scale_b, shift_b, 0, 0}, nseq = (M - 1) / seq + 1;
    for (int i = 0; i < 5; ++i) {
        auto meets = [&](const void *out, int64_t ldo, int64_t n, int64_t rows) {
            return rows_share_vectors(out, ldo, n, rows, vectors[i], steps[i], nseq, D);
        };
        ok = ok && !meets(h_out, ldho, D, M) && !(z_scales ? meets(z, pad * D / 2, pad * D / 2, 1) || meets(z_scales, pad * D / 64, pad * D / 64, 1)
                                                           : meets(z, ldz, D, M));
    }
    QIM_REQUIRE(ok, QIM_ERR_ARG, "%s: an output overlaps an input other than as the same rows, or the other output", who);
    ResNormArgs a{(const uint16_t *)h, (const uint16_t *)x, (const uint16_t *)post_weight, (const uint16_t *)gate,
                  (const uint16_t *)norm_weight, (const uint16_t *)scale, (const uint16_t *)shift, (uint16_t *)h_out,
                  z_scales ? nullptr : (uint16_t *)z, z_scales ? (uint8_t *)z : nullptr, (uint8_t *)z_scales, ldh, ldx, ldho, ldz,
                  gate_b, scale_b, shift_b, M, pad, (int)D, post, norm, (flags & QIM_ADALN_ADD_ONE) ? 1 : 0,
                  (flags & QIM_ADALN_TILED) ? 1 : 0, (uint32_t)seq, alpha, post_eps, norm_eps, 1.0 / (double)D};
    hipStream_t st = as_stream(stream);
    if (z_scales) {
        if (eager) launch_residual_norm<true, true>(a, st);
        else launch_residual_norm<true, false>(a, st);
    } else {
        if (eager) launch_residual_norm<false, true>(a, st);
        else launch_residual_norm<false, false>(a, st);
    }
    return check_launch(who);
}
