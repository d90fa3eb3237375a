// Backward of the residual update between two norms: the kernel (mathematics, bound and the types' roles: resnorm.hip), in E channels a lane;
// a source file of its own compiles each width.
//
// Column sums (the vectors' gradients, a per-sample gate's) stay in registers over all rows of a workgroup: eight channels a lane, up to 48
// accumulators, which is what limits a lane to one chunk; the vectors themselves are read from LDS.  A workgroup walks UNITS: rows of
// one sample, so a per-sample gate's gradient is flushed once a unit.  Partial sums of the workgroups are joined by a second, small
// launch in a fixed order; nothing is atomic.  An accumulator adds one term for each row that its lane takes, in 32 bits: at most
// rows / (workgroups x rows at once) of them, 4096 for 2^20 rows of 4096 channels, then 48 + 32 in the join (up to 1536 workgroups).
#pragma once
#include "resnorm.h"

struct ResnormBwdArgs {
    const void *dh, *dy, *h, *b, *gate;               // one that is not given points at another of its type: it is loaded for nothing, from the cache
    int has_dh, has_dy;
    void *dx, *db, *dgate;                            // dgate: per row
    const float* stats;
    const float *post_w, *post_b, *scale, *keep, *pre_w;
    float *partial, *gate_partial;                    // [blocks][slots][C] column sums; [units][C] of the per-sample gate, none where a unit is a sample
    int lddh, lddy, ldh, ldb, ldg;
    int sample_rows;                                  // rows that `units_per_sample` units cover: one sample's where the gate is per sample, else all
    FastDiv per_sample;
    int units, units_per_sample, slots, ragged;       // ragged 1: some lane owns nothing; 2: one owns less than eight channels
    int C, lpr, post, pre, gate_mode, act;
    float alpha;
};

// Slots of `partial`, in this order, those that exist: pre weight, pre bias, post weight, post bias, scale.
template <typename D> __device__ __forceinline__ void put(void* dst, int i, float v, bool as_d) { if (as_d) ((D*)dst)[i] = from_f<D>(v); else ((float*)dst)[i] = v; }
template <int WAVES, typename D = float, int E> __device__ __forceinline__ void flush_columns(float (&acc)[E], void* dst, bool as_d, int C, Cols k, int lpr, float* sh) {
    k = here(k);
    if constexpr (WAVES > 1) {                                               // a thread owns its columns; two hold the same of those they share
        if (k.lo < E) {
            if (as_d) {
                Chunk<D, E> t;
#pragma unroll
                for (int e = 0; e < E; ++e) t.set(e, acc[e]);
                t.store((D*)dst + k.cb);
            } else {
                Chunk<float, E> t;
#pragma unroll
                for (int e = 0; e < E; ++e) t.set(e, acc[e]);
                t.store((float*)dst + k.cb);
            }
        }
    } else {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int e = 0; e < E; ++e) for (int o = lpr; o < 64; o <<= 1) acc[e] += __shfl_xor(acc[e], o, 64);
        __syncthreads();                                                     // the previous flush has been read
        if (lane < lpr) {
#pragma unroll
            for (int e = 0; e < E; ++e) if (e >= k.lo) sh[(threadIdx.x >> 6) * 512 + k.cb + e] = acc[e];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < C; i += 256) put<D>(dst, i, (sh[i] + sh[512 + i]) + (sh[1024 + i] + sh[1536 + i]), as_d);
    }
}

template <typename TX, typename TB, int E, bool GATE> struct BwdRow { Chunk<TX, E> dh, h; Chunk<TB, E> dy, b, g[1]; float keep; floatx4 st; };

// Waves a SIMD, which bounds the registers (512 / waves); the grid is what is resident then: a second, partial round of workgroups would
// run at a fraction of the waves.  bf16 without a post norm or gate: four, which is between (join included, 16 x 65536 x 64 174 us, three 167;
// 65536 x 320 50, three 53; 65536 x 384 58, three 57).  Rows that several waves share in eights, bf16: one less, for fewer partial sums
// (LN + LN + gate, 24 M elements, C = 1024 81 -> 68 us; in sixes it would cost, 640 73 -> 81).
__host__ __device__ constexpr int bwd_waves(int width, int waves, bool narrow, bool post, int gate) {
    if (waves > 4) return 2;
    if (narrow && waves > 1 && width == 8) return post ? 2 : 3;
    // an f32 stream around bf16 does not fit three waves' registers here, and f32 around f32 is no slower with two (24 M elements, RMS behind:
    // C = 1024 129 -> 124 us, 2048 126 -> 122)
    if (!narrow && waves > 1 && width == 8 && gate == 1) return 2;
    return narrow ? (!post && gate == 0 ? 4 : 3) : post ? 2 : 3;
}

// Measured (sizes as at the forward): 176 us = 4.7 TB/s, 63 us = 4.8, 142 us = 5.2; the join behind it 4 to 5 us.
template <typename TX, typename TB, int E, int WAVES, bool POST, int GATE>
__global__ __launch_bounds__(WAVES > 1 ? WAVES * 64 : 256, bwd_waves(E, WAVES, sizeof(TX) == 2, POST, GATE)) void resnorm_bwd_kernel(ResnormBwdArgs a) {
    constexpr int THREADS = WAVES > 1 ? WAVES * 64 : 256;
    extern __shared__ __attribute__((aligned(16))) float vec[];              // post weight | post bias | scale | pre weight
    __shared__ float sh[WAVES > 1 ? 4 * WAVES : 4 * 512];
    int turn = 0;
    const int lpr = WAVES > 1 ? THREADS : a.lpr, lane = threadIdx.x & 63, lig = WAVES > 1 ? (int)threadIdx.x : lane & (lpr - 1), lanes = WAVES > 1 ? 64 : lpr;
    const int rpw = WAVES > 1 ? 1 : 64 / lpr;
    const int lr = WAVES > 1 ? 0 : lane / lpr, groups = WAVES > 1 ? 1 : 4 * rpw;   // this lane's row among the wave's; rows a workgroup takes at once
    const int wave_first = WAVES > 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * rpw;
    const Cols k = cols_of<E>(lig * E, a.C);
    const float invC = 1.f / a.C;
    const int vlen = lpr * E;
    // A thread that owns its columns fetches its chunk of every vector, otherwise a wave fetches a vector: one latency, not one for every 256
    // values (LN + LN + gate in bf16, 24 M elements: C = 768 79 -> 70 us, 4096 83 -> 69; wide rows with a gate in a f32 stream 155 -> 147)
    if constexpr (WAVES > 1) {
        float w[4][E];
        load_vec(w[0], a.post_w, 1.f, k); load_vec(w[1], a.post_b, 0.f, k); load_vec(w[2], a.scale, 1.f, k); load_vec(w[3], a.pre_w, 1.f, k);
#pragma unroll
        for (int i = 0; i < 4; ++i) put_chunk(vec + i * vlen, w[i], lig, lpr);
    } else if (lane < lpr) {
        const int i = threadIdx.x >> 6;
        float w[E];
        load_vec(w, i == 0 ? a.post_w : i == 1 ? a.post_b : i == 2 ? a.scale : a.pre_w, i == 1 ? 0.f : 1.f, k);
        put_chunk(vec + i * vlen, w, lig, lpr);
    }
    __syncthreads();
    auto sums = [&](const float (&g)[E], const float (&hat)[E], float& s1, float& s2) {      // a channel counts once
        if (a.ragged == 2) {
            const Cols own = here(k);
#pragma unroll
            for (int e = 0; e < E; ++e) { const float v = e < own.lo ? 0.f : g[e]; s1 += v; s2 = fmaf(v, hat[e], s2); }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) { s1 += g[e]; s2 = fmaf(g[e], hat[e], s2); }
            if (a.ragged && lig * E >= a.C) { s1 = 0.f; s2 = 0.f; }
        }
    };
    float dwp[E] = {}, dbp[E] = {}, dwq[E] = {}, dbq[E] = {}, dsc[E] = {}, dgs[E] = {};
    for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        // a unit: every units_per_sample-th step of a sample's rows, so that the workgroups at work read one stretch of memory together
        // (a contiguous share each puts thousands of streams a power of two apart: MiT stage 1 210 -> 203 us)
        const int smp_u = unit / a.units_per_sample;
        const int begin = smp_u * a.sample_rows, end = begin + a.sample_rows;
        const int start = (unit - smp_u * a.units_per_sample) * groups, stride = a.units_per_sample * groups;
        Chunk<TB, E> unit_gate;
        if constexpr (GATE == 1) unit_gate.load(at<TB>(a.gate, smp_u, a.ldg, (unsigned)k.cb));
        // as the forward: two rows of registers, and the same number of steps for everybody who shares a row sum
        auto load = [&](BwdRow<TX, TB, E, GATE == 2>& t, int i) {
            const int row = begin + wave_first + i < end ? begin + wave_first + i : end - 1;   // the wave's first row
            const unsigned l = row + lr < end ? (unsigned)lr : 0u, cb = (unsigned)k.cb;
            t.keep = a.keep ? a.keep[GATE == 1 ? (unsigned)smp_u : fdiv((unsigned)row + l, a.per_sample)] : 1.f;
            t.dy.load(at<TB>(a.dy, row, a.lddy, l * (unsigned)a.lddy + cb));
            t.h.load(at<TX>(a.h, row, a.ldh, l * (unsigned)a.ldh + cb));
            t.dh.load(at<TX>(a.dh, row, a.lddh, l * (unsigned)a.lddh + cb));
            t.b.load(at<TB>(a.b, row, a.ldb, l * (unsigned)a.ldb + cb));
            if constexpr (GATE == 2) t.g[0].load(at<TB>(a.gate, row, a.ldg, l * (unsigned)a.ldg + cb));
            t.st = *at<floatx4>(a.stats, row, 1, l);
        };
        auto work = [&](BwdRow<TX, TB, E, GATE == 2>& t, int i) {
            const int row = begin + wave_first + i;
            const bool there = row + lr < end, ok = there && k.lo < E;
            const unsigned dense = (unsigned)(lr * a.C + k.cb);
            if (row + rpw > end && !there) {                                 // a lane without a row adds nothing to the columns, infinities neither
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    t.dy.set(e, 0.f); t.dh.set(e, 0.f); t.h.set(e, 0.f); t.b.set(e, 0.f);
                    if constexpr (GATE == 2) t.g[0].set(e, 0.f);
                }
                t.st = floatx4{0.f, 0.f, 0.f, 0.f};
            }
                float d[E], hat[E], v[E];
                if (a.has_dh) {
#pragma unroll
                    for (int e = 0; e < E; ++e) d[e] = t.dh.get(e);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) d[e] = 0.f;
                }
                if (a.has_dy) {                                              // through the norm behind h
                    const float mh = t.st[2], rh = t.st[3];
                    float g[E], s1 = 0.f, s2 = 0.f;
                    vec_chunk(v, vec + 3 * vlen, lig, lpr);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float gy = t.dy.get(e);
                        hat[e] = (t.h.get(e) - mh) * rh;
                        dwp[e] = fmaf(gy, hat[e], dwp[e]); dbp[e] += gy;
                        g[e] = gy * v[e];
                    }
                    sums(g, hat, s1, s2);
                    row_sum2<WAVES>(s1, s2, lanes, sh, turn);
                    s1 = a.pre == 1 ? s1 * invC : 0.f; s2 *= invC;
#pragma unroll
                    for (int e = 0; e < E; ++e) d[e] = fmaf(rh, fmaf(-hat[e], s2, g[e] - s1), d[e]);
                }
                if (ok) {
                    Chunk<TX, E> o;
#pragma unroll
                    for (int e = 0; e < E; ++e) o.set(e, d[e] * a.alpha);
                    o.store(at((TX*)a.dx, row, a.C, dense));
                }
                // dn, the scale's and the gate's gradients; n = hat w + bias
                float act[E], nn[E];
                const float mu = t.st[0], r = t.st[1];
                if (a.keep) {
#pragma unroll
                    for (int e = 0; e < E; ++e) d[e] *= t.keep;
                }
                if constexpr (POST) {
                    float w[E];
                    vec_chunk(w, vec, lig, lpr); vec_chunk(v, vec + vlen, lig, lpr);
#pragma unroll
                    for (int e = 0; e < E; ++e) { hat[e] = (t.b.get(e) - mu) * r; nn[e] = fmaf(hat[e], w[e], v[e]); }
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) nn[e] = t.b.get(e);
                }
                vec_chunk(v, vec + 2 * vlen, lig, lpr);
#pragma unroll
                for (int e = 0; e < E; ++e) nn[e] *= d[e];
                if constexpr (GATE != 0) {
                    const Chunk<TB, E>& g = GATE == 1 ? unit_gate : t.g[0];
                    if (a.act) {
#pragma unroll
                        for (int e = 0; e < E; ++e) act[e] = sigmoid_f(g.get(e));
                    } else {
#pragma unroll
                        for (int e = 0; e < E; ++e) act[e] = g.get(e);
                    }
#pragma unroll
                    for (int e = 0; e < E; ++e) { dsc[e] = fmaf(nn[e], act[e], dsc[e]); d[e] *= v[e] * act[e]; nn[e] *= v[e]; }
                    if (a.act) {
#pragma unroll
                        for (int e = 0; e < E; ++e) nn[e] *= fmaf(-act[e], act[e], act[e]);
                    }
                    if constexpr (GATE == 1) {
#pragma unroll
                        for (int e = 0; e < E; ++e) dgs[e] += nn[e];
                    } else if (ok) {
                        Chunk<TB, E> o;
#pragma unroll
                        for (int e = 0; e < E; ++e) o.set(e, nn[e]);
                        o.store(at((TB*)a.dgate, row, a.C, dense));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) { dsc[e] += nn[e]; d[e] *= v[e]; }
                }
                if constexpr (POST) {                                        // through the norm of b
                    float s1 = 0.f, s2 = 0.f;
                    vec_chunk(v, vec, lig, lpr);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        dwq[e] = fmaf(d[e], hat[e], dwq[e]); dbq[e] += d[e];
                        d[e] *= v[e];
                    }
                    sums(d, hat, s1, s2);
                    row_sum2<WAVES>(s1, s2, lanes, sh, turn);
                    s1 = a.post == 1 ? s1 * invC : 0.f; s2 *= invC;
#pragma unroll
                    for (int e = 0; e < E; ++e) d[e] = r * fmaf(-hat[e], s2, d[e] - s1);
                }
                if (ok) {
                    Chunk<TB, E> o;
#pragma unroll
                    for (int e = 0; e < E; ++e) o.set(e, d[e]);
                    o.store(at((TB*)a.db, row, a.C, dense));
                }
        };
        BwdRow<TX, TB, E, GATE == 2> r0, r1;
        load(r0, start);
        for (int i = start; begin + wave_first + i < end; i += 2 * stride) {
            asm volatile("" ::: "memory");                                   // the vectors stay in LDS
            load(r1, i + stride);
            work(r0, i);
            if (begin + wave_first + i + stride >= end) break;
            asm volatile("" ::: "memory");
            load(r0, i + 2 * stride);
            work(r1, i + stride);
        }
        if constexpr (GATE == 1) {
            // to the partial sums, or to the gradient itself where the unit is the sample
            flush_columns<WAVES, TB>(dgs, a.gate_partial ? (void*)(a.gate_partial + (int64_t)unit * a.C) : (void*)((TB*)a.dgate + (int64_t)smp_u * a.C),
                                     !a.gate_partial, a.C, k, lpr, sh);
#pragma unroll
            for (int e = 0; e < E; ++e) dgs[e] = 0.f;
        }
    }
    float* dst = a.partial + (int64_t)blockIdx.x * a.slots * a.C;
    if (a.pre) { flush_columns<WAVES>(dwp, dst, false, a.C, k, lpr, sh); dst += a.C; }
    if (a.pre == 1) { flush_columns<WAVES>(dbp, dst, false, a.C, k, lpr, sh); dst += a.C; }
    if constexpr (POST) {
        flush_columns<WAVES>(dwq, dst, false, a.C, k, lpr, sh); dst += a.C;
        if (a.post == 1) { flush_columns<WAVES>(dbq, dst, false, a.C, k, lpr, sh); dst += a.C; }
    }
    if (a.scale) flush_columns<WAVES>(dsc, dst, false, a.C, k, lpr, sh);
}

// Workgroups of the launch: waves of a row, lanes of a row of less than a wave, workgroups
struct ResnormLaunch { int x_dtype, b_dtype, waves, lpr, blocks; };
template <int E> static void resnorm_bwd_launch(const ResnormBwdArgs& a, const ResnormLaunch& p, hipStream_t stream) {
    const size_t shm = (size_t)4 * (p.waves > 1 ? p.waves * 64 : p.lpr) * E * sizeof(float);
#define SS_RN_L(TX, TB, W, P, G) hipLaunchKernelGGL((resnorm_bwd_kernel<TX, TB, E, W, P, G>), dim3((unsigned)p.blocks), dim3(W > 1 ? W * 64 : 256), shm, stream, a)
#define SS_RN_G(TX, TB, W, P) do { if (a.gate_mode == 0) SS_RN_L(TX, TB, W, P, 0); else if (a.gate_mode == 1) SS_RN_L(TX, TB, W, P, 1); \
        else SS_RN_L(TX, TB, W, P, 2); } while (0)
#define SS_RN_P(TX, TB, W) do { if (a.post) SS_RN_G(TX, TB, W, true); else SS_RN_G(TX, TB, W, false); } while (0)
#define SS_RN_W(TX, TB) do { switch (p.waves) { case 1: SS_RN_P(TX, TB, 1); break; case 2: SS_RN_P(TX, TB, 2); break; \
        case 4: SS_RN_P(TX, TB, 4); break; default: SS_RN_P(TX, TB, 8); } } while (0)
    if constexpr (E == 1) {
        if (p.x_dtype == SS_BF16) SS_RN_P(bf16, bf16, 1); else if (p.b_dtype == SS_BF16) SS_RN_P(float, bf16, 1); else SS_RN_P(float, float, 1);
    } else if (p.x_dtype == SS_BF16) SS_RN_W(bf16, bf16); else if (p.b_dtype == SS_BF16) SS_RN_W(float, bf16); else SS_RN_W(float, float);
#undef SS_RN_L
#undef SS_RN_G
#undef SS_RN_P
#undef SS_RN_W
}
void resnorm_bwd_launch6(const ResnormBwdArgs& a, const ResnormLaunch& p, hipStream_t stream);
void resnorm_bwd_launch1(const ResnormBwdArgs& a, const ResnormLaunch& p, hipStream_t stream);
