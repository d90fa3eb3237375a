// The residual update between two blocks with a norm on either side of it, forward and backward.
//
// Mathematics, per row r of sample s = r / rows_per_sample, over C channels:
//   n = post(b)                                       none, LayerNorm (w, bias) or RMSNorm (w)
//   h = alpha x + keep[s] scale[c] act(gate) n        gate per sample or per row; act: identity or sigmoid
//   y = pre(h)                                        over h AS STORED (rounded to the stream's type): what every reader of h sees
// backward, with hhat and nhat the normalised rows, m() the mean over the row (0 where RMSNorm has no mean to remove):
//   dH = dh + r_h (g - m(g) - hhat m(g hhat)),  g = dy w_pre;         dx = alpha dH
//   dn = dH keep scale act(gate);               db = r_b (g' - m(g') - nhat m(g' nhat)),  g' = dn w_post
//   dgate = dH keep scale n act'(gate);         dscale, dw, dbias: column sums over the rows
//
// Bound by HBM: x, b (, gate) in, h, y out; backward dh, dy, h, b (, gate) and 16 bytes of statistics a row in, dx, db (, dgate) out.
// So everything between the two norms happens in registers, a row is read once, and its four statistics are kept for the backward
// (recomputing them there would cost two more reductions a row and save 16 bytes).
//
// Work split: a row is a power of two of lanes with 8 channels each.  Up to 512 channels a wave holds 64 / lanes rows; above, the WAVES
// of a workgroup share the row and join their sums through LDS.  Row sums are taken in double, sum and sum of squares in ONE pass: the
// variance does not cancel (double holds the square of any float exactly), one reduction serves mean and variance, and the result is
// the same to the last bit of a float whatever the split -- h is rounded to 8 bits behind it, and an h near the border of two values
// would otherwise depend on the order of a sum.  Products and sums up to h are rounded one by one (no contraction) for the same reason.
#include "common.h"

struct ResnormArgs {
    const void *x, *b, *gate;
    void *h, *y;
    float* stats;                                     // [rows][4]: mean, 1 / deviation of b; the same of h
    const float *post_w, *post_b, *scale, *keep, *pre_w, *pre_b;
    int64_t ldx, ldb, ldg;
    int64_t rows;
    FastDiv per_sample;                               // rows of one sample
    int C, lpr, post, pre, gate_mode, act;            // norms: 0 none, 1 LayerNorm, 2 RMSNorm; gate: 0 none, 1 per sample, 2 per row
    float alpha;
    double eps;
};

struct ResnormBwdArgs {
    const void *dh, *dy, *h, *b, *gate;
    void *dx, *db, *dgate;                            // dgate: per row
    const float* stats;
    const float *post_w, *post_b, *scale, *keep, *pre_w;
    float *partial, *gate_partial;                    // [blocks][slots][C] column sums; [units][C] of the per-sample gate
    int64_t lddh, lddy, ldh, ldb, ldg;
    int64_t rows, unit_rows;                          // a unit: consecutive rows of ONE sample (of all rows where the gate is not per sample)
    int64_t sample_rows;                              // rows that `units_per_sample` units cover
    FastDiv per_sample;
    int units, units_per_sample, slots;
    int C, lpr, post, pre, gate_mode, act;
    float alpha;
};

// ---------------------------------------------------------------- eight channels of a row
// Row starts need no alignment beyond the element's (odd widths, odd row strides): global memory takes the access as one.
struct __attribute__((packed, aligned(2))) Bf8u { bf16x8 v; };
struct __attribute__((packed, aligned(4))) Fl8u { floatx4 a, b; };
template <typename T> struct Chunk;
template <> struct Chunk<bf16> {
    bf16x8 v;
    __device__ __forceinline__ void load(const bf16* p) { v = ((const Bf8u*)p)->v; }
    __device__ __forceinline__ float get(int e) const { return (float)v[e]; }
    __device__ __forceinline__ void set(int e, float f) { v[e] = (bf16)f; }
    __device__ __forceinline__ void store(bf16* p) const { ((Bf8u*)p)->v = v; }
};
template <> struct Chunk<float> {
    floatx4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = ((const Fl8u*)p)->a; b = ((const Fl8u*)p)->b; }
    __device__ __forceinline__ float get(int e) const { return e < 4 ? a[e & 3] : b[e & 3]; }
    __device__ __forceinline__ void set(int e, float f) { if (e < 4) a[e & 3] = f; else b[e & 3] = f; }
    __device__ __forceinline__ void store(float* p) const { ((Fl8u*)p)->a = a; ((Fl8u*)p)->b = b; }
};
// n: channels left from here on (a lane past the row's end has none)
template <typename T> __device__ __forceinline__ void load_chunk(Chunk<T>& c, const T* p, int n) {
    if (n >= 8) { c.load(p); return; }
#pragma unroll
    for (int e = 0; e < 8; ++e) c.set(e, e < n ? to_f(p[e]) : 0.f);
}
template <typename T> __device__ __forceinline__ void store_chunk(const Chunk<T>& c, T* p, int n) {
    if (n >= 8) { c.store(p); return; }
#pragma unroll
    for (int e = 0; e < 7; ++e) if (e < n) p[e] = from_f<T>(c.get(e));
}
__device__ __forceinline__ void load_vec(float (&v)[8], const float* p, int c, int n, float otherwise) {
    if (p && n >= 8) { const Fl8u* q = (const Fl8u*)(p + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = q->a[e]; v[4 + e] = q->b[e]; }
        return; }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = p && e < n ? p[c + e] : otherwise;
}

// ---------------------------------------------------------------- row sums
template <int CTRL> __device__ __forceinline__ double dpp_add_d(double v) {
    const long long u = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xf, 0xf, true);
    return v + __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
}
__device__ __forceinline__ double dgroup_sum(double v, int lanes) {         // over aligned groups of a power of two of lanes
    if (lanes >= 2) v = dpp_add_d<0xB1>(v);
    if (lanes >= 4) v = dpp_add_d<0x4E>(v);
    if (lanes >= 8) v = dpp_add_d<0x141>(v);
    if (lanes >= 16) v = dpp_add_d<0x140>(v);
    for (int o = 16; o < lanes; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// Two sums over the lanes of a row.  `sh` has two halves used in turn: a wave may enter the next sum while another still reads this one,
// but not the one after it.
template <int WAVES, typename S> __device__ __forceinline__ void row_sum2(S& a, S& b, int lanes, S* sh, int& turn) {
    if constexpr (sizeof(S) == 8) { a = dgroup_sum(a, lanes); b = dgroup_sum(b, lanes); }
    else { a = group_sum(a, lanes); b = group_sum(b, lanes); }
    if constexpr (WAVES > 1) {
        S* s = sh + turn * 2 * WAVES;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) { s[(threadIdx.x >> 6) * 2] = a; s[(threadIdx.x >> 6) * 2 + 1] = b; }
        __syncthreads();
        a = s[0]; b = s[1];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) { a += s[w * 2]; b += s[w * 2 + 1]; }
    }
}
// 1 / sqrt(x) from v_rsq_f64 (about 26 bits) and one Newton step
__device__ __forceinline__ double rsqrt_d(double x) {
    const double y = __builtin_amdgcn_rsq(x);
    return y * fma(-0.5 * x * y, y, 1.5);
}
template <int WAVES> __device__ __forceinline__ void row_stats(double s, double q, int kind, int C, double eps, int lanes, double* sh, int& turn, float& mu, float& r) {
    row_sum2<WAVES>(s, q, lanes, sh, turn);
    const double inv = 1.0 / (double)C, m = kind == 1 ? s * inv : 0.0;
    double var = fma(-m, m, q * inv);
    var = var > 0.0 ? var : (var < 0.0 ? 0.0 : var);                        // NaN stays
    mu = (float)m; r = (float)rsqrt_d(var + eps);
}
__device__ __forceinline__ float sigmoid_f(float v) { return __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

// ---------------------------------------------------------------- forward
template <typename TX, typename TB, int WAVES, int U>
__global__ __launch_bounds__(WAVES > 1 ? WAVES * 64 : 256) void resnorm_fwd_kernel(ResnormArgs a) {
#pragma clang fp contract(off)
    __shared__ double sh[WAVES > 1 ? 4 * WAVES : 1];
    int turn = 0;
    const int lane = threadIdx.x & 63, lig = WAVES > 1 ? (int)threadIdx.x : lane & (a.lpr - 1), lanes = WAVES > 1 ? 64 : a.lpr;
    const int rpw = WAVES > 1 ? 1 : 64 / a.lpr;
    const int64_t group = WAVES > 1 ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * rpw + lane / a.lpr;
    const int64_t groups = WAVES > 1 ? (int64_t)gridDim.x : (int64_t)gridDim.x * 4 * rpw;
    const int c = lig * 8, n = a.C - c;
    float wq[8], bq[8], sc[8], wp[8], bp[8];
    load_vec(wq, a.post_w, c, n, 1.f); load_vec(bq, a.post_b, c, n, 0.f); load_vec(sc, a.scale, c, n, 1.f);
    load_vec(wp, a.pre_w, c, n, 1.f); load_vec(bp, a.pre_b, c, n, 0.f);
    // all lanes of a wave (all waves of a workgroup that shares a row) walk the same number of steps: the row sums are joint
    const int64_t first = WAVES > 1 ? group : group - lane / a.lpr;
    for (int64_t r0 = 0; first + r0 < a.rows; r0 += U * groups) {
        Chunk<TX> xv[U];
        Chunk<TB> bv[U], gv[U];
        int64_t row[U];
        float kp[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            row[u] = group + r0 + u * groups;
            const int k = row[u] < a.rows ? n : 0;
            const int64_t rr = row[u] < a.rows ? row[u] : 0;
            load_chunk(xv[u], (const TX*)a.x + rr * a.ldx + c, k);
            load_chunk(bv[u], (const TB*)a.b + rr * a.ldb + c, k);
            const int64_t smp = fdiv((unsigned)rr, a.per_sample);
            if (a.gate_mode) load_chunk(gv[u], (const TB*)a.gate + (a.gate_mode == 1 ? smp : rr) * a.ldg + c, k);
            kp[u] = a.keep ? a.keep[smp] : 1.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (WAVES > 1 && row[u] >= a.rows) break;                        // the same for the whole workgroup
            const int k = row[u] < a.rows ? n : 0;
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = bv[u].get(e);
            float mu = 0.f, r = 0.f, mh = 0.f, rh = 0.f;
            if (a.post) {
                double s = 0.0, q = 0.0;
#pragma unroll
                for (int e = 0; e < 8; ++e) { const double d = (double)f[e]; s += d; q = __builtin_fma(d, d, q); }
                row_stats<WAVES>(s, q, a.post, a.C, a.eps, lanes, sh, turn, mu, r);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = (f[e] - mu) * r * wq[e] + bq[e];
            }
            if (a.gate_mode) {
#pragma unroll
                for (int e = 0; e < 8; ++e) { const float g = gv[u].get(e); f[e] *= a.act ? sigmoid_f(g) : g; }
            }
            if (a.scale) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= sc[e];
            }
            if (a.keep) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= kp[u];
            }
            Chunk<TX> hv;
#pragma unroll
            for (int e = 0; e < 8; ++e) hv.set(e, xv[u].get(e) * a.alpha + f[e]);
            if (k > 0) store_chunk(hv, (TX*)a.h + row[u] * a.C + c, k);
            if (a.pre) {
                double s = 0.0, q = 0.0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f[e] = e < k ? hv.get(e) : 0.f;                          // what lies past the row's end is no part of its sums
                    const double d = (double)f[e]; s += d; q = __builtin_fma(d, d, q);
                }
                row_stats<WAVES>(s, q, a.pre, a.C, a.eps, lanes, sh, turn, mh, rh);
                if (k > 0) {
                    Chunk<TB> yv;
#pragma unroll
                    for (int e = 0; e < 8; ++e) yv.set(e, (f[e] - mh) * rh * wp[e] + bp[e]);
                    store_chunk(yv, (TB*)a.y + row[u] * a.C + c, k);
                }
            }
            if (a.stats && lig == 0 && row[u] < a.rows) *(floatx4*)(a.stats + row[u] * 4) = floatx4{mu, r, mh, rh};
        }
    }
}

// ---------------------------------------------------------------- backward
// Column sums stay in registers over all rows of a workgroup; the per-sample gate's are flushed at the end of each unit.
// Slots of `partial`, in this order, those that exist: pre weight, pre bias, post weight, post bias, scale.
template <int WAVES> __device__ __forceinline__ void flush_columns(float (&acc)[8], float* __restrict__ dst, int C, int c, int n, int lpr, float* sh) {
    if constexpr (WAVES > 1) {                                               // a thread owns its columns
#pragma unroll
        for (int e = 0; e < 8; ++e) if (e < n) dst[c + e] = acc[e];
    } else {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int e = 0; e < 8; ++e) for (int o = lpr; o < 64; o <<= 1) acc[e] += __shfl_xor(acc[e], o, 64);
        __syncthreads();                                                     // the previous flush has been read
        if (lane < lpr) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sh[(threadIdx.x >> 6) * 512 + c + e] = acc[e];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < C; i += 256) dst[i] = (sh[i] + sh[512 + i]) + (sh[1024 + i] + sh[1536 + i]);
    }
}

template <typename TX, typename TB, int WAVES, int U>
__global__ __launch_bounds__(WAVES > 1 ? WAVES * 64 : 256) void resnorm_bwd_kernel(ResnormBwdArgs a) {
    __shared__ float sh[WAVES > 1 ? 4 * WAVES : 4 * 512];
    int turn = 0;
    const int lane = threadIdx.x & 63, lig = WAVES > 1 ? (int)threadIdx.x : lane & (a.lpr - 1), lanes = WAVES > 1 ? 64 : a.lpr;
    const int rpw = WAVES > 1 ? 1 : 64 / a.lpr;
    const int group = WAVES > 1 ? 0 : (threadIdx.x >> 6) * rpw + lane / a.lpr, groups = WAVES > 1 ? 1 : 4 * rpw;
    const int wave_first = WAVES > 1 ? 0 : (threadIdx.x >> 6) * rpw;
    const int c = lig * 8, n = a.C - c;
    const float invC = 1.f / a.C;
    float wq[8], bq[8], sc[8], wp[8];
    load_vec(wq, a.post_w, c, n, 1.f); load_vec(bq, a.post_b, c, n, 0.f); load_vec(sc, a.scale, c, n, 1.f); load_vec(wp, a.pre_w, c, n, 1.f);
    float dwp[8] = {}, dbp[8] = {}, dwq[8] = {}, dbq[8] = {}, dsc[8] = {}, dgs[8] = {};
    for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const int smp_u = unit / a.units_per_sample;
        const int64_t begin = (int64_t)smp_u * a.sample_rows + (int64_t)(unit - smp_u * a.units_per_sample) * a.unit_rows;
        const int64_t stop = (int64_t)(smp_u + 1) * a.sample_rows;
        const int64_t end = begin + a.unit_rows < stop ? begin + a.unit_rows : stop;
        for (int64_t r0 = begin; r0 + wave_first < end; r0 += U * groups) {
            Chunk<TX> dhv[U], hv[U];
            Chunk<TB> dyv[U], bv[U], gv[U];
            int64_t row[U];
            float kp[U];
            floatx4 st[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                row[u] = r0 + u * groups + group;
                const int k = row[u] < end ? n : 0;
                const int64_t rr = row[u] < end ? row[u] : begin;
                if (a.dh) load_chunk(dhv[u], (const TX*)a.dh + rr * a.lddh + c, k);
                if (a.dy) load_chunk(dyv[u], (const TB*)a.dy + rr * a.lddy + c, k);
                if (a.dy) load_chunk(hv[u], (const TX*)a.h + rr * a.ldh + c, k);
                load_chunk(bv[u], (const TB*)a.b + rr * a.ldb + c, k);
                const int64_t smp = fdiv((unsigned)rr, a.per_sample);
                if (a.gate_mode) load_chunk(gv[u], (const TB*)a.gate + (a.gate_mode == 1 ? smp : rr) * a.ldg + c, k);
                kp[u] = a.keep ? a.keep[smp] : 1.f;
                st[u] = *(const floatx4*)(a.stats + rr * 4);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (WAVES > 1 && row[u] >= end) break;                       // the same for the whole workgroup
                const int k = row[u] < end ? n : 0;
                float d[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = a.dh ? dhv[u].get(e) : 0.f;
                if (a.dy) {                                                  // through the norm behind h
                    const float mh = st[u][2], rh = st[u][3];
                    float g[8], hh[8], s1 = 0.f, s2 = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float t = dyv[u].get(e);                       // zero past the row's end, with everything that follows from it
                        hh[e] = e < k ? (hv[u].get(e) - mh) * rh : 0.f;
                        dwp[e] = fmaf(t, hh[e], dwp[e]); dbp[e] += t;
                        g[e] = t * wp[e];
                        s1 += g[e]; s2 = fmaf(g[e], hh[e], s2);
                    }
                    row_sum2<WAVES>(s1, s2, lanes, sh, turn);
                    s1 = a.pre == 1 ? s1 * invC : 0.f; s2 *= invC;
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] += rh * (g[e] - s1 - hh[e] * s2);
                }
                if (k > 0) {
                    Chunk<TX> o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o.set(e, d[e] * a.alpha);
                    store_chunk(o, (TX*)a.dx + row[u] * a.C + c, k);
                }
                const float mu = st[u][0], r = st[u][1];
                float nh[8], dg[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    d[e] = e < k ? d[e] * kp[u] : 0.f;
                    nh[e] = e < k ? (a.post ? (bv[u].get(e) - mu) * r : bv[u].get(e)) : 0.f;
                    const float nn = a.post ? fmaf(nh[e], wq[e], bq[e]) : nh[e];
                    float act = 1.f, slope = 1.f;
                    if (a.gate_mode) { act = gv[u].get(e); if (a.act) { act = sigmoid_f(act); slope = act * (1.f - act); } }
                    const float dn = d[e] * nn;
                    dsc[e] = fmaf(dn, act, dsc[e]);
                    dg[e] = dn * sc[e] * slope;
                    dgs[e] += dg[e];
                    d[e] *= sc[e] * act;
                }
                if (a.gate_mode == 2 && k > 0) {
                    Chunk<TB> o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o.set(e, dg[e]);
                    store_chunk(o, (TB*)a.dgate + row[u] * a.C + c, k);
                }
                if (a.post) {                                                // through the norm of b
                    float s1 = 0.f, s2 = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        dwq[e] = fmaf(d[e], nh[e], dwq[e]); dbq[e] += d[e];
                        d[e] *= wq[e];
                        s1 += d[e]; s2 = fmaf(d[e], nh[e], s2);
                    }
                    row_sum2<WAVES>(s1, s2, lanes, sh, turn);
                    s1 = a.post == 1 ? s1 * invC : 0.f; s2 *= invC;
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] = r * (d[e] - s1 - nh[e] * s2);
                }
                if (k > 0) {
                    Chunk<TB> o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o.set(e, d[e]);
                    store_chunk(o, (TB*)a.db + row[u] * a.C + c, k);
                }
            }
        }
        if (a.gate_mode == 1) {
            flush_columns<WAVES>(dgs, a.gate_partial + (int64_t)unit * a.C, a.C, c, n, a.lpr, sh);
#pragma unroll
            for (int e = 0; e < 8; ++e) dgs[e] = 0.f;
        }
    }
    float* dst = a.partial + (int64_t)blockIdx.x * a.slots * a.C;
    if (a.pre) { flush_columns<WAVES>(dwp, dst, a.C, c, n, a.lpr, sh); dst += a.C; }
    if (a.pre == 1) { flush_columns<WAVES>(dbp, dst, a.C, c, n, a.lpr, sh); dst += a.C; }
    if (a.post) { flush_columns<WAVES>(dwq, dst, a.C, c, n, a.lpr, sh); dst += a.C; }
    if (a.post == 1) { flush_columns<WAVES>(dbq, dst, a.C, c, n, a.lpr, sh); dst += a.C; }
    if (a.scale) flush_columns<WAVES>(dsc, dst, a.C, c, n, a.lpr, sh);
}

// Joins the partial sums in a fixed order: workgroup row blockIdx.x < slots is a vector's gradient, the others are samples' gates.
// 8 columns x 32 parts a workgroup, as colreduce_final_kernel.
template <typename TB>
__global__ __launch_bounds__(256) void resnorm_join_kernel(const float* __restrict__ partial, int blocks, int slots, float* __restrict__ out,
        const float* __restrict__ gate_partial, int units_per_sample, TB* __restrict__ dgate, int C) {
    __shared__ float sh[32][9];
    const int cx = threadIdx.x & 7, part = threadIdx.x >> 3, col = blockIdx.y * 8 + cx;
    const bool vec = (int)blockIdx.x < slots;
    const int smp = (int)blockIdx.x - slots;
    const float* p = vec ? partial + (int64_t)blockIdx.x * C : gate_partial + (int64_t)smp * units_per_sample * C;
    const int64_t step = vec ? (int64_t)slots * C : C;
    const int count = vec ? blocks : units_per_sample;
    float s = 0.f;
    if (col < C) {
#pragma unroll 4
        for (int i = part; i < count; i += 32) s += p[(int64_t)i * step + col];
    }
    sh[part][cx] = s;
    __syncthreads();
    if (part == 0 && col < C) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += sh[i][cx];
        if (vec) out[(int64_t)blockIdx.x * C + col] = t; else dgate[(int64_t)smp * C + col] = from_f<TB>(t);
    }
}

// ---------------------------------------------------------------- C ABI
#define SS_RESNORM_MAX_C 4096
static int waves_of(int C) { return C <= 512 ? 1 : C <= 1024 ? 2 : C <= 2048 ? 4 : 8; }
static int lanes_of(int C) { int l = 1; while (l * 8 < C && l < 64) l <<= 1; return l; }

static int resnorm_check(const char* who, int x_dtype, int b_dtype, int64_t rows, int64_t rows_per_sample, int C, int post, int pre, int gate_mode,
                         int act, const void* gate, const float* post_w, const float* post_b, const float* pre_w, const float* pre_b, bool biases) {
    SS_CHECK((x_dtype == SS_F32 && (b_dtype == SS_F32 || b_dtype == SS_BF16)) || (x_dtype == SS_BF16 && b_dtype == SS_BF16),
             "%s: stream / branch types must be f32 / f32, bf16 / bf16 or f32 / bf16, got codes %d / %d", who, x_dtype, b_dtype);
    SS_CHECK(rows > 0 && rows < (1LL << 31) && rows_per_sample > 0 && rows % rows_per_sample == 0, "%s: bad row counts (%lld, %lld a sample)", who,
             (long long)rows, (long long)rows_per_sample);
    SS_CHECK(C > 0 && C <= SS_RESNORM_MAX_C, "%s: C=%d must be 1 to %d", who, C, SS_RESNORM_MAX_C);
    SS_CHECK(post >= 0 && post <= 2 && pre >= 0 && pre <= 2 && gate_mode >= 0 && gate_mode <= 2 && act >= 0 && act <= 1, "%s: bad codes", who);
    SS_CHECK((gate_mode != 0) == (gate != nullptr), "%s: a gate and its layout go together", who);
    SS_CHECK((!post || post_w) && (!pre || pre_w), "%s: a norm needs its weight", who);
    SS_CHECK(!biases || ((post == 1 || !post_b) && (pre == 1 || !pre_b)), "%s: only LayerNorm takes a bias", who);
    return 0;
}

#define SS_RESNORM_LAUNCH(KERNEL, TX, TB, W, U, GRID, ARGS) \
    hipLaunchKernelGGL((KERNEL<TX, TB, W, U>), dim3((unsigned)(GRID)), dim3(W > 1 ? W * 64 : 256), 0, stream, ARGS)
#define SS_RESNORM_WAVES(KERNEL, TX, TB, WAVES, GRID, ARGS) do { switch (WAVES) { \
        case 1: SS_RESNORM_LAUNCH(KERNEL, TX, TB, 1, 2, GRID, ARGS); break; \
        case 2: SS_RESNORM_LAUNCH(KERNEL, TX, TB, 2, 2, GRID, ARGS); break; \
        case 4: SS_RESNORM_LAUNCH(KERNEL, TX, TB, 4, 2, GRID, ARGS); break; \
        default: SS_RESNORM_LAUNCH(KERNEL, TX, TB, 8, 1, GRID, ARGS); } } while (0)
#define SS_RESNORM_TYPES(KERNEL, WAVES, GRID, ARGS) do { \
        if (x_dtype == SS_BF16) SS_RESNORM_WAVES(KERNEL, bf16, bf16, WAVES, GRID, ARGS); \
        else if (b_dtype == SS_BF16) SS_RESNORM_WAVES(KERNEL, float, bf16, WAVES, GRID, ARGS); \
        else SS_RESNORM_WAVES(KERNEL, float, float, WAVES, GRID, ARGS); } while (0)

extern "C" int ss_resnorm_fwd(int x_dtype, int b_dtype, const void* x, int64_t ldx, const void* b, int64_t ldb, const void* gate, int64_t ldg, int gate_mode,
                              int act, const float* scale, const float* keep, float alpha, int post, const float* post_w, const float* post_b, int pre,
                              const float* pre_w, const float* pre_b, double eps, void* h, void* y, float* stats, int64_t rows, int64_t rows_per_sample,
                              int C, hipStream_t stream) {
    if (gate_mode == 1 && rows_per_sample == 1) gate_mode = 2;               // a sample of one row
    if (int rc = resnorm_check("ss_resnorm_fwd", x_dtype, b_dtype, rows, rows_per_sample, C, post, pre, gate_mode, act, gate, post_w, post_b, pre_w, pre_b, true)) return rc;
    SS_CHECK(x && b && h && (!pre || y) && ldx >= 0 && ldb >= 0 && ldg >= 0 && eps >= 0.0, "ss_resnorm_fwd: bad arguments");
    ResnormArgs a;
    a.x = x; a.b = b; a.gate = gate; a.h = h; a.y = y; a.stats = stats; a.post_w = post_w; a.post_b = post_b; a.scale = scale; a.keep = keep;
    a.pre_w = pre_w; a.pre_b = pre_b; a.ldx = ldx; a.ldb = ldb; a.ldg = ldg; a.rows = rows; a.per_sample = fast_div((unsigned)rows_per_sample);
    a.C = C; a.lpr = lanes_of(C); a.post = post; a.pre = pre; a.gate_mode = gate_mode; a.act = act; a.alpha = alpha; a.eps = eps;
    const int waves = waves_of(C);
    const int64_t rows_per_wg = waves > 1 ? 1 : 4 * (64 / a.lpr), want = cdiv(rows, rows_per_wg), most = waves > 1 ? 16384 / waves : 4096;
    const int64_t grid = want < most ? want : most;
    SS_RESNORM_TYPES(resnorm_fwd_kernel, waves, grid, a);
    SS_LAUNCH_CHECK();
    return 0;
}

struct ResnormPlan { int waves, lpr, slots, blocks, units, units_per_sample; int64_t unit_rows, sample_rows; };
static ResnormPlan resnorm_plan(int64_t rows, int64_t rows_per_sample, int C, int post, int pre, int gate_mode, bool scale) {
    ResnormPlan p;
    p.waves = waves_of(C); p.lpr = lanes_of(C);
    p.slots = (pre ? 1 : 0) + (pre == 1 ? 1 : 0) + (post ? 1 : 0) + (post == 1 ? 1 : 0) + (scale ? 1 : 0);
    p.sample_rows = gate_mode == 1 ? rows_per_sample : rows;
    const int64_t samples = rows / p.sample_rows;
    const int64_t most = p.waves > 1 ? 4096 / p.waves : 1024;                // workgroups
    const int64_t step = p.waves > 1 ? 1 : 4 * (64 / p.lpr);                 // rows a workgroup takes at once
    int64_t per = most / samples;                                            // units of a sample: enough for all workgroups, each of at least one step
    if (per > cdiv(p.sample_rows, step)) per = cdiv(p.sample_rows, step);
    if (per < 1) per = 1;
    p.unit_rows = cdiv(cdiv(p.sample_rows, per), step) * step;
    p.units_per_sample = (int)cdiv(p.sample_rows, p.unit_rows);
    const int64_t units = samples * p.units_per_sample;
    p.units = (int)units;
    p.blocks = (int)(units < most ? units : most);
    return p;
}

extern "C" int64_t ss_resnorm_bwd_workspace(int64_t rows, int64_t rows_per_sample, int C, int post, int pre, int gate_mode, int has_scale) {
    if (rows <= 0 || rows_per_sample <= 0 || C <= 0 || C > SS_RESNORM_MAX_C || rows >= (1LL << 31)) return 0;
    if (gate_mode == 1 && rows_per_sample == 1) gate_mode = 2;
    const ResnormPlan p = resnorm_plan(rows, rows_per_sample, C, post, pre, gate_mode, has_scale != 0);
    return ((int64_t)p.blocks * p.slots + (gate_mode == 1 ? p.units : 0)) * C * 4;
}

extern "C" int ss_resnorm_bwd(int x_dtype, int b_dtype, const void* dh, int64_t lddh, const void* dy, int64_t lddy, const void* h, int64_t ldh,
                              const void* b, int64_t ldb, const void* gate, int64_t ldg, int gate_mode, int act, const float* scale, const float* keep,
                              float alpha, int post, const float* post_w, const float* post_b, int pre, const float* pre_w, const float* stats, void* dx,
                              void* db, void* dgate, float* dvec, int64_t rows, int64_t rows_per_sample, int C, float* workspace, int64_t ws_bytes,
                              hipStream_t stream) {
    if (gate_mode == 1 && rows_per_sample == 1) gate_mode = 2;               // a sample of one row
    if (int rc = resnorm_check("ss_resnorm_bwd", x_dtype, b_dtype, rows, rows_per_sample, C, post, pre, gate_mode, act, gate, post_w, post_b, pre_w, nullptr, false)) return rc;
    SS_CHECK(b && stats && dx && db && (dh || dy) && (!dy || (pre && h)) && (!gate || dgate) && lddh >= 0 && lddy >= 0 && ldh >= 0 && ldb >= 0 && ldg >= 0,
             "ss_resnorm_bwd: bad arguments");
    const ResnormPlan p = resnorm_plan(rows, rows_per_sample, C, post, pre, gate_mode, scale != nullptr);
    const int64_t need = ((int64_t)p.blocks * p.slots + (gate_mode == 1 ? p.units : 0)) * C * 4;
    SS_CHECK((p.slots == 0 || dvec) && (need == 0 || (workspace && ws_bytes >= need)), "ss_resnorm_bwd: workspace too small (%lld of %lld bytes)",
             (long long)ws_bytes, (long long)need);
    ResnormBwdArgs a;
    a.dh = dh; a.dy = dy; a.h = h; a.b = b; a.gate = gate; a.dx = dx; a.db = db; a.dgate = dgate; a.stats = stats; a.post_w = post_w; a.post_b = post_b;
    a.scale = scale; a.keep = keep; a.pre_w = pre_w; a.partial = workspace; a.gate_partial = workspace + (int64_t)p.blocks * p.slots * C;
    a.lddh = lddh; a.lddy = lddy; a.ldh = ldh; a.ldb = ldb; a.ldg = ldg; a.rows = rows; a.unit_rows = p.unit_rows; a.sample_rows = p.sample_rows;
    a.per_sample = fast_div((unsigned)rows_per_sample); a.units = p.units; a.units_per_sample = p.units_per_sample; a.slots = p.slots;
    a.C = C; a.lpr = p.lpr; a.post = post; a.pre = pre; a.gate_mode = gate_mode; a.act = act; a.alpha = alpha;
    SS_RESNORM_TYPES(resnorm_bwd_kernel, p.waves, p.blocks, a);
    SS_LAUNCH_CHECK();
    const int64_t join = p.slots + (gate_mode == 1 ? rows / rows_per_sample : 0);
    if (join > 0) {
        const dim3 grid((unsigned)join, (unsigned)cdiv(C, 8));
        if (b_dtype == SS_BF16) hipLaunchKernelGGL(resnorm_join_kernel<bf16>, grid, dim3(256), 0, stream, workspace, p.blocks, p.slots, dvec,
                                                   a.gate_partial, p.units_per_sample, (bf16*)dgate, C);
        else hipLaunchKernelGGL(resnorm_join_kernel<float>, grid, dim3(256), 0, stream, workspace, p.blocks, p.slots, dvec, a.gate_partial,
                                p.units_per_sample, (float*)dgate, C);
        SS_LAUNCH_CHECK();
    }
    return 0;
}
