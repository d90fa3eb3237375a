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
#include "resnorm.h"

struct ResnormArgs {
    const void *x, *b, *gate;
    void *h, *y;
    float* stats;                                     // [rows][4]: mean, 1 / deviation of b; the same of h
    const float *post_w, *post_b, *scale, *keep, *pre_w, *pre_b;
    int ldx, ldb, ldg, rows;
    FastDiv per_sample;                               // rows of one sample
    double inv_c;
    int ragged;                                       // 1: some lane owns nothing; 2: one owns less than eight channels
    int C, lpr, post, pre, gate_mode, act;            // norms: 0 none, 1 LayerNorm, 2 RMSNorm; gate: 0 none, 1 per sample, 2 per row
    float alpha;
    double eps;
};

// One lane's part of a row: NCH chunks of 8 channels
template <typename TX, typename TB, int NCH, bool GATE> struct FwdRow { Chunk<TX> x[NCH]; Chunk<TB> b[NCH], g[GATE ? NCH : 1]; float keep; };

template <typename TX, typename TB, int WAVES, int NCH, bool POST, int GATE>   // GATE: 0 none, 1 per sample, 2 per row
__global__ __launch_bounds__(WAVES > 1 ? WAVES * 64 : 256) void resnorm_fwd_kernel(ResnormArgs a) {
#pragma clang fp contract(off)
    constexpr int THREADS = WAVES > 1 ? WAVES * 64 : 256;
    extern __shared__ __attribute__((aligned(16))) float vec[];              // WAVES == 1: post weight | post bias | scale | pre weight | pre bias
    __shared__ double sh[WAVES > 1 ? 4 * WAVES : 1];
    int turn = 0;
    const int lpr = WAVES > 1 ? THREADS : a.lpr, lane = threadIdx.x & 63, lig = WAVES > 1 ? (int)threadIdx.x : lane & (lpr - 1), lanes = WAVES > 1 ? 64 : lpr;
    const int chunks = lpr * NCH, rpw = WAVES > 1 ? 1 : 64 / lpr;
    const int lr = WAVES > 1 ? 0 : lane / lpr;                               // this lane's row among the wave's
    const int first = WAVES > 1 ? (int)blockIdx.x : ((int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)) * rpw;
    const int groups = WAVES > 1 ? (int)gridDim.x : (int)gridDim.x * 4 * rpw;

    auto load = [&](FwdRow<TX, TB, NCH, GATE != 0>& t, int i) {
        const int row = first + i < a.rows ? first + i : a.rows - 1;     // the wave's first row; past the end the last one, for nothing
        const unsigned l = row + lr < a.rows ? (unsigned)lr : 0u;
        const unsigned smp = a.keep || GATE == 1 ? fdiv((unsigned)row + l, a.per_sample) : 0u;
        t.keep = a.keep ? a.keep[smp] : 1.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const unsigned cb = (unsigned)cols_of((lig + j * lpr) * 8, a.C).cb;
            load_chunk(t.b[j], at<TB>(a.b, row, a.ldb, l * (unsigned)a.ldb + cb), a.C);
            if constexpr (GATE == 1) load_chunk(t.g[j], (const TB*)a.gate + (int64_t)smp * a.ldg + cb, a.C);
            if constexpr (GATE == 2) load_chunk(t.g[j], at<TB>(a.gate, row, a.ldg, l * (unsigned)a.ldg + cb), a.C);
            load_chunk(t.x[j], at<TX>(a.x, row, a.ldx, l * (unsigned)a.ldx + cb), a.C);
        }
    };
    FwdRow<TX, TB, NCH, GATE != 0> r0;
    load(r0, 0);                                                             // on its way while the vectors are fetched
    // The vectors: a thread of a row that takes a whole workgroup owns its columns and keeps them in registers (80 KB of LDS would leave one
    // workgroup a CU and cost more to fill than four rows to read); a wave with several rows reads them from LDS, one copy for all rows
    // (in registers they would take 40 a chunk).
    const int vlen = chunks * 8;
    float own[WAVES > 1 ? 5 : 1][8];
    if constexpr (WAVES > 1) {
        const Cols k = cols_of(lig * 8, a.C);
        load_vec(own[0], a.post_w, 1.f, k); load_vec(own[1], a.post_b, 0.f, k); load_vec(own[2], a.scale, 1.f, k);
        load_vec(own[3], a.pre_w, 1.f, k); load_vec(own[4], a.pre_b, 0.f, k);
    } else {
        if (POST) { stage_vec(vec, a.post_w, 1.f, a.C, chunks, THREADS); stage_vec(vec + vlen, a.post_b, 0.f, a.C, chunks, THREADS); }
        if (a.scale) stage_vec(vec + 2 * vlen, a.scale, 1.f, a.C, chunks, THREADS);
        if (a.pre) { stage_vec(vec + 3 * vlen, a.pre_w, 1.f, a.C, chunks, THREADS); stage_vec(vec + 4 * vlen, a.pre_b, 0.f, a.C, chunks, THREADS); }
        __syncthreads();
    }
    auto vector = [&](float (&v)[8], int which, int j) {
        if constexpr (WAVES > 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = own[which][e];
        } else vec_chunk(v, vec + which * vlen, lig + j * lpr, chunks);
    };
    auto sums = [&](const float (&f)[NCH][8], double& s, double& q) {        // a channel counts once
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            double cs = 0.0, cq = 0.0;
            if (a.ragged == 2) {
                const Cols k = here(cols_of((lig + j * lpr) * 8, a.C));
#pragma unroll
                for (int e = 0; e < 8; ++e) { const float v = e < k.lo || e >= k.hi ? 0.f : f[j][e]; const double d = (double)v; cs += d; cq = __builtin_fma(d, d, cq); }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) { const double d = (double)f[j][e]; cs += d; cq = __builtin_fma(d, d, cq); }
                if (a.ragged && (lig + j * lpr) * 8 >= a.C) { cs = 0.0; cq = 0.0; }
            }
            s += cs; q += cq;
        }
    };
    auto work = [&](const FwdRow<TX, TB, NCH, GATE != 0>& t, int i) {
#pragma clang fp contract(off)
        const int row = first + i;
        const bool ok = row + lr < a.rows;
        float f[NCH][8], v[8];
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) f[j][e] = t.b[j].get(e);
            float mu = 0.f, r = 0.f, mh = 0.f, rh = 0.f;
            if constexpr (POST) {
                double s = 0.0, q = 0.0;
                sums(f, s, q);
                row_stats<WAVES>(s, q, a.post, a.inv_c, a.eps, lanes, sh, turn, mu, r);
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    vector(v, 0, j);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[j][e] = (f[j][e] - mu) * r * v[e];
                    if (a.post_b) {
                        vector(v, 1, j);
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[j][e] += v[e];
                    }
                }
            }
            if constexpr (GATE != 0) {
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    if (a.act) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[j][e] *= sigmoid_f(t.g[j].get(e));
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[j][e] *= t.g[j].get(e);
                    }
                }
            }
            if (a.scale) {
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    vector(v, 2, j);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[j][e] *= v[e];
                }
            }
            if (a.keep) {
#pragma unroll
                for (int j = 0; j < NCH; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[j][e] *= t.keep;
            }
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                const Cols k = cols_of((lig + j * lpr) * 8, a.C);
                Chunk<TX> hv;
#pragma unroll
                for (int e = 0; e < 8; ++e) hv.set(e, t.x[j].get(e) * a.alpha + f[j][e]);
                if (ok && k.lo < k.hi) store_chunk(hv, at((TX*)a.h, row, a.C, (unsigned)(lr * a.C + k.cb)), a.C);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[j][e] = hv.get(e);
            }
            if (a.pre) {
                double s = 0.0, q = 0.0;
                sums(f, s, q);
                row_stats<WAVES>(s, q, a.pre, a.inv_c, a.eps, lanes, sh, turn, mh, rh);
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    const Cols k = cols_of((lig + j * lpr) * 8, a.C);
                    float w[8];
                    vector(w, 3, j); vector(v, 4, j);
                    Chunk<TB> yv;
#pragma unroll
                    for (int e = 0; e < 8; ++e) yv.set(e, (f[j][e] - mh) * rh * w[e] + v[e]);
                    if (ok && k.lo < k.hi) store_chunk(yv, at((TB*)a.y, row, a.C, (unsigned)(lr * a.C + k.cb)), a.C);
                }
            }
        if (a.stats && lig == 0 && ok) *at((floatx4*)a.stats, row, 1, (unsigned)lr) = floatx4{mu, r, mh, rh};
    };
    // All lanes of a wave (all waves of a workgroup that shares a row) walk the same number of steps: the row sums are joint.  Up to two
    // chunks a lane there are two rows of registers, the next row on its way while this one is worked on; with more, two rows would leave a
    // SIMD one wave, and the other waves' loads do the same.
    if constexpr (NCH <= 2) {
        FwdRow<TX, TB, NCH, GATE != 0> r1;
        for (int i = 0; first + i < a.rows; i += 2 * groups) {
            asm volatile("" ::: "memory");                                   // the vectors stay in LDS
            load(r1, i + groups);
            work(r0, i);
            if (first + i + groups >= a.rows) break;
            asm volatile("" ::: "memory");
            load(r0, i + 2 * groups);
            work(r1, i + groups);
        }
    } else {
        for (int i = 0; first + i < a.rows; i += groups) {
            asm volatile("" ::: "memory");
            work(r0, i);
            load(r0, i + groups);
        }
    }
}

// ---------------------------------------------------------------- C ABI
extern "C" int ss_resnorm_fwd(int x_dtype, int b_dtype, const void* x, int64_t ldx, const void* b, int64_t ldb, const void* gate, int64_t ldg, int gate_mode,
                              int act, const float* scale, const float* keep, float alpha, int post, const float* post_w, const float* post_b, int pre,
                              const float* pre_w, const float* pre_b, double eps, void* h, void* y, float* stats, int64_t rows, int64_t rows_per_sample,
                              int C, hipStream_t stream) {
    if (gate_mode == 1 && rows_per_sample == 1) gate_mode = 2;               // a sample of one row
    if (int rc = resnorm_check("ss_resnorm_fwd", x_dtype, b_dtype, rows, rows_per_sample, C, post, pre, gate_mode, act, gate, post_w, post_b, pre_w, pre_b, true)) return rc;
    SS_CHECK(x && b && h && (!pre || y) && ldx >= 0 && ldb >= 0 && ldg >= 0 && ldx < SS_RESNORM_MAX_LD && ldb < SS_RESNORM_MAX_LD &&
             ldg < SS_RESNORM_MAX_LD && eps >= 0.0, "ss_resnorm_fwd: bad arguments");
    ResnormArgs a;
    a.x = x; a.b = b; a.gate = gate; a.h = h; a.y = y; a.stats = stats; a.post_w = post_w; a.post_b = post_b; a.scale = scale; a.keep = keep;
    a.pre_w = pre_w; a.pre_b = pre_b; a.ldx = (int)ldx; a.ldb = (int)ldb; a.ldg = (int)ldg; a.rows = (int)rows; a.per_sample = fast_div((unsigned)rows_per_sample);
    a.C = C; a.post = post; a.pre = pre; a.gate_mode = gate_mode; a.act = act; a.alpha = alpha; a.eps = eps; a.inv_c = 1.0 / (double)C;
    const int chunks = (int)cdiv(C, 8);
    int waves = 1, nch = 1;
    // Lanes of a row, measured at 24 M elements:
    // - a stream in 32 bits is bound by its bytes: one chunk a lane, whole lines in a load (C = 96: 85 us, 96 in four lanes, 100 in eight;
    //   320: 80 in 64 lanes, 103 in sixteen), above 512 channels 32 lanes (768: 96, 106 in 64);
    // - a bf16 stream with norms and gates is bound by vector instructions: up to four chunks a lane so that the fewest lanes are idle, of those
    //   the most lanes (C = 96 in 4 x 3: 44 us, 53 in 16; 384 in 16 x 3: 43, 57 in 64; 128 in 16: 41, 43 in 8 x 2);
    // - with rows too few for a wave on every SIMD, as many lanes as there are chunks (1 row of 512: 6.4 -> 5.0 us).
    const bool wide = x_dtype == SS_F32 || rows * chunks < 64 * 1024;
    if (chunks <= 64 && wide) { a.lpr = 1; while (a.lpr < chunks) a.lpr <<= 1; }
    else if (chunks <= 128) {
        int slots = 1 << 30;
        for (int l = x_dtype == SS_F32 && rows * chunks >= 64 * 1024 ? 32 : 64; l >= 1; l >>= 1) {
            const int n = (int)cdiv(chunks, l);
            if (n <= 4 && l * n < slots) { slots = l * n; a.lpr = l; nch = n; }
        }
    }
    else { waves = chunks <= 256 ? 4 : 8; a.lpr = waves * 64; }
    a.ragged = C % 8 ? 2 : C != a.lpr * nch * 8;
    const int64_t want = waves > 1 ? rows : cdiv(rows, 4 * (64 / a.lpr)), most = waves > 1 ? 4096 / waves : 1024;
    const unsigned grid = (unsigned)(want < most ? want : most);
    const size_t shm = waves > 1 ? 0 : (size_t)5 * a.lpr * nch * 8 * sizeof(float);
#define SS_RN_L(TX, TB, W, N, P, G) hipLaunchKernelGGL((resnorm_fwd_kernel<TX, TB, W, N, P, G>), dim3(grid), dim3(W > 1 ? W * 64 : 256), shm, stream, a)
#define SS_RN_GATE(TX, TB, W, N, P) do { if (gate_mode == 0) SS_RN_L(TX, TB, W, N, P, 0); else if (gate_mode == 1) SS_RN_L(TX, TB, W, N, P, 1); \
        else SS_RN_L(TX, TB, W, N, P, 2); } while (0)
#define SS_RN_PG(TX, TB, W, N) do { if (post) SS_RN_GATE(TX, TB, W, N, true); else SS_RN_GATE(TX, TB, W, N, false); } while (0)
#define SS_RN_G(TX, TB) do { if (waves == 8) SS_RN_PG(TX, TB, 8, 1); else if (waves == 4) SS_RN_PG(TX, TB, 4, 1); \
        else if (nch == 4) SS_RN_PG(TX, TB, 1, 4); else if (nch == 3) SS_RN_PG(TX, TB, 1, 3); else if (nch == 2) SS_RN_PG(TX, TB, 1, 2); \
        else SS_RN_PG(TX, TB, 1, 1); } while (0)
    if (x_dtype == SS_BF16) SS_RN_G(bf16, bf16); else if (b_dtype == SS_BF16) SS_RN_G(float, bf16); else SS_RN_G(float, float);
    SS_LAUNCH_CHECK();
    return 0;
}
