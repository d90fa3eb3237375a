// Forward of the residual update between two norms: the kernel (mathematics and work split: resnorm.hip), in E channels a chunk; a source file
// of its own compiles each width.
#pragma once
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

// One lane's part of a row: NCH chunks of E channels
template <typename TX, typename TB, int E, int NCH, bool GATE> struct FwdRow { Chunk<TX, E> x[NCH]; Chunk<TB, E> b[NCH], g[GATE ? NCH : 1]; float keep; };

// Measured: 16 x 65536 x 64 in bf16, one norm: 97 us = 5.5 TB/s (a copy runs at 5.0); 65536 x 384 in bf16, two LayerNorms, a gate: 49 us =
// 4.1 TB/s, bound by vector instructions; 8192 x 4096, a f32 stream around bf16, two RMSNorms, a gate per row: 87 us = 5.4 TB/s; one row
// of 512: 3.6 us, a launch.
template <typename TX, typename TB, int E, int WAVES, int NCH, bool POST, int GATE>   // GATE: 0 none, 1 per sample, 2 per row
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

    auto load = [&](FwdRow<TX, TB, E, NCH, GATE != 0>& t, int i) {
        const int row = first + i < a.rows ? first + i : a.rows - 1;     // the wave's first row; past the end the last one, for nothing
        const unsigned l = row + lr < a.rows ? (unsigned)lr : 0u;
        const unsigned smp = a.keep || GATE == 1 ? fdiv((unsigned)row + l, a.per_sample) : 0u;
        t.keep = a.keep ? a.keep[smp] : 1.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const unsigned cb = (unsigned)cols_of<E>((lig + j * lpr) * E, a.C).cb;
            t.b[j].load(at<TB>(a.b, row, a.ldb, l * (unsigned)a.ldb + cb));
            if constexpr (GATE == 1) t.g[j].load((const TB*)a.gate + (int64_t)smp * a.ldg + cb);
            if constexpr (GATE == 2) t.g[j].load(at<TB>(a.gate, row, a.ldg, l * (unsigned)a.ldg + cb));
            t.x[j].load(at<TX>(a.x, row, a.ldx, l * (unsigned)a.ldx + cb));
        }
    };
    FwdRow<TX, TB, E, NCH, GATE != 0> r0;
    load(r0, 0);                                                             // on its way while the vectors are fetched
    // The vectors: a thread of a row that takes a whole workgroup owns its columns and keeps them in registers (80 KB of LDS would leave one
    // workgroup a CU and cost more to fill than four rows to read); a wave with several rows reads them from LDS, one copy for all rows
    // (in registers they would take 40 a chunk).
    const int vlen = chunks * E;
    float own[WAVES > 1 ? 5 : 1][E];
    if constexpr (WAVES > 1) {
        const Cols k = cols_of<E>(lig * E, a.C);
        load_vec(own[0], a.post_w, 1.f, k); load_vec(own[1], a.post_b, 0.f, k); load_vec(own[2], a.scale, 1.f, k);
        load_vec(own[3], a.pre_w, 1.f, k); load_vec(own[4], a.pre_b, 0.f, k);
    } else {
        // a wave fetches a vector (the first one two), every chunk of it in flight at once
        const int w = threadIdx.x >> 6;
        if (lane < lpr) {
            float v[NCH][E], u[NCH][E];
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                const Cols k = cols_of<E>((lig + j * lpr) * E, a.C);
                load_vec(v[j], w == 0 ? a.post_w : w == 1 ? a.post_b : w == 2 ? a.scale : a.pre_w, w == 1 ? 0.f : 1.f, k);
                if (w == 0) load_vec(u[j], a.pre_b, 0.f, k);
            }
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                put_chunk(vec + w * vlen, v[j], lig + j * lpr, chunks);
                if (w == 0) put_chunk(vec + 4 * vlen, u[j], lig + j * lpr, chunks);
            }
        }
        __syncthreads();
    }
    auto vector = [&](float (&v)[E], int which, int j) {
        if constexpr (WAVES > 1) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = own[which][e];
        } else vec_chunk(v, vec + which * vlen, lig + j * lpr, chunks);
    };
    auto sums = [&](const float (&f)[NCH][E], double& s, double& q) {        // a channel counts once
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            double cs = 0.0, cq = 0.0;
            if (a.ragged == 2) {
                const Cols k = here(cols_of<E>((lig + j * lpr) * E, a.C));
#pragma unroll
                for (int e = 0; e < E; ++e) { const float v = e < k.lo ? 0.f : f[j][e]; const double d = (double)v; cs += d; cq = __builtin_fma(d, d, cq); }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) { const double d = (double)f[j][e]; cs += d; cq = __builtin_fma(d, d, cq); }
                if (a.ragged && (lig + j * lpr) * E >= a.C) { cs = 0.0; cq = 0.0; }
            }
            s += cs; q += cq;
        }
    };
    auto work = [&](const FwdRow<TX, TB, E, NCH, GATE != 0>& t, int i) {
#pragma clang fp contract(off)
        const int row = first + i;
        const bool ok = row + lr < a.rows;
        float f[NCH][E], v[E];
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) f[j][e] = t.b[j].get(e);
            float mu = 0.f, r = 0.f, mh = 0.f, rh = 0.f;
            if constexpr (POST) {
                double s = 0.0, q = 0.0;
                sums(f, s, q);
                row_stats<WAVES>(s, q, a.post, a.inv_c, a.eps, lanes, sh, turn, mu, r);
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    vector(v, 0, j);
#pragma unroll
                    for (int e = 0; e < E; ++e) f[j][e] = (f[j][e] - mu) * r * v[e];
                    if (a.post_b) {
                        vector(v, 1, j);
#pragma unroll
                        for (int e = 0; e < E; ++e) f[j][e] += v[e];
                    }
                }
            }
            if constexpr (GATE != 0) {
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    if (a.act) {
#pragma unroll
                        for (int e = 0; e < E; ++e) f[j][e] *= sigmoid_f(t.g[j].get(e));
                    } else {
#pragma unroll
                        for (int e = 0; e < E; ++e) f[j][e] *= t.g[j].get(e);
                    }
                }
            }
            if (a.scale) {
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    vector(v, 2, j);
#pragma unroll
                    for (int e = 0; e < E; ++e) f[j][e] *= v[e];
                }
            }
            if (a.keep) {
#pragma unroll
                for (int j = 0; j < NCH; ++j)
#pragma unroll
                    for (int e = 0; e < E; ++e) f[j][e] *= t.keep;
            }
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                const Cols k = cols_of<E>((lig + j * lpr) * E, a.C);
                Chunk<TX, E> hv;
#pragma unroll
                for (int e = 0; e < E; ++e) hv.set(e, t.x[j].get(e) * a.alpha + f[j][e]);
                if (ok && k.lo < E) hv.store(at((TX*)a.h, row, a.C, (unsigned)(lr * a.C + k.cb)));
#pragma unroll
                for (int e = 0; e < E; ++e) f[j][e] = hv.get(e);
            }
            if (a.pre) {
                double s = 0.0, q = 0.0;
                sums(f, s, q);
                row_stats<WAVES>(s, q, a.pre, a.inv_c, a.eps, lanes, sh, turn, mh, rh);
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    const Cols k = cols_of<E>((lig + j * lpr) * E, a.C);
                    float w[E];
                    vector(w, 3, j); vector(v, 4, j);
                    Chunk<TB, E> yv;
#pragma unroll
                    for (int e = 0; e < E; ++e) yv.set(e, (f[j][e] - mh) * rh * w[e] + v[e]);
                    if (ok && k.lo < E) yv.store(at((TB*)a.y, row, a.C, (unsigned)(lr * a.C + k.cb)));
                }
            }
        if (a.stats && lig == 0 && ok) *at((floatx4*)a.stats, row, 1, (unsigned)lr) = floatx4{mu, r, mh, rh};
    };
    // All lanes of a wave (all waves of a workgroup that shares a row) walk the same number of steps: the row sums are joint.  Up to two
    // chunks a lane there are two rows of registers, the next row on its way while this one is worked on; with more, two rows would leave a
    // SIMD one wave, and the other waves' loads do the same.
    if constexpr (NCH <= 2) {
        FwdRow<TX, TB, E, NCH, GATE != 0> r1;
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

// six channels: a bf16 stream whose rows take several waves; one: rows of less than eight
struct ResnormFwdLaunch { int x_dtype, b_dtype, waves, nch, blocks; };
template <int E> static void resnorm_fwd_launch(const ResnormArgs& a, const ResnormFwdLaunch& p, hipStream_t stream) {
    const size_t shm = p.waves > 1 ? 0 : (size_t)5 * a.lpr * p.nch * E * sizeof(float);
#define SS_RN_L(TX, TB, W, N, P, G) hipLaunchKernelGGL((resnorm_fwd_kernel<TX, TB, E, W, N, P, G>), dim3((unsigned)p.blocks), dim3(W > 1 ? W * 64 : 256), shm, stream, a)
#define SS_RN_GATE(TX, TB, W, N, P) do { if (a.gate_mode == 0) SS_RN_L(TX, TB, W, N, P, 0); else if (a.gate_mode == 1) SS_RN_L(TX, TB, W, N, P, 1); \
        else SS_RN_L(TX, TB, W, N, P, 2); } while (0)
#define SS_RN_PG(TX, TB, W, N) do { if (a.post) SS_RN_GATE(TX, TB, W, N, true); else SS_RN_GATE(TX, TB, W, N, false); } while (0)
#define SS_RN_W(TX, TB) do { if (p.waves == 8) SS_RN_PG(TX, TB, 8, 1); else if (p.waves == 4) SS_RN_PG(TX, TB, 4, 1); else SS_RN_PG(TX, TB, 2, 1); } while (0)
    if constexpr (E == 1) {
        if (p.x_dtype == SS_BF16) SS_RN_PG(bf16, bf16, 1, 1); else if (p.b_dtype == SS_BF16) SS_RN_PG(float, bf16, 1, 1); else SS_RN_PG(float, float, 1, 1);
    } else if constexpr (E == 6) SS_RN_W(bf16, bf16);
    else if (p.waves > 1) { if (p.x_dtype == SS_BF16) SS_RN_W(bf16, bf16); else if (p.b_dtype == SS_BF16) SS_RN_W(float, bf16); else SS_RN_W(float, float); }
    else if (p.x_dtype == SS_F32) { if (p.b_dtype == SS_F32) SS_RN_PG(float, float, 1, 1); else SS_RN_PG(float, bf16, 1, 1); }
    else if (p.nch == 4) SS_RN_PG(bf16, bf16, 1, 4);                         // only a bf16 stream takes more than one chunk a lane
    else if (p.nch == 3) SS_RN_PG(bf16, bf16, 1, 3);
    else if (p.nch == 2) SS_RN_PG(bf16, bf16, 1, 2);
    else SS_RN_PG(bf16, bf16, 1, 1);
#undef SS_RN_L
#undef SS_RN_GATE
#undef SS_RN_PG
#undef SS_RN_W
}
void resnorm_fwd_launch6(const ResnormArgs& a, const ResnormFwdLaunch& p, hipStream_t stream);
void resnorm_fwd_launch1(const ResnormArgs& a, const ResnormFwdLaunch& p, hipStream_t stream);
