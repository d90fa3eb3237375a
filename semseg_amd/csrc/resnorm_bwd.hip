// Backward of the residual update between two norms (mathematics, bound and the types' roles: resnorm.hip).
//
// Column sums (the vectors' gradients, a per-sample gate's) stay in registers over all rows of a workgroup: eight channels a lane, up to 48
// accumulators, which is what limits a lane to one chunk; the vectors themselves are read from LDS.  A workgroup walks UNITS: rows of
// one sample, so a per-sample gate's gradient is flushed once a unit.  Partial sums of the workgroups are joined by a second, small
// launch in a fixed order; nothing is atomic.
#include "resnorm.h"

struct __attribute__((packed, aligned(4))) Fl4u { floatx4 v; };

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
template <int WAVES, typename D = float> __device__ __forceinline__ void flush_columns(float (&acc)[8], void* dst, bool as_d, int C, Cols k, int lpr, float* sh) {
    k = here(k);
    if constexpr (WAVES > 1) {                                               // a thread owns its columns
#pragma unroll
        for (int e = 0; e < 8; ++e) if (e >= k.lo && e < k.hi) put<D>(dst, k.cb + e, acc[e], as_d);
    } else {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int e = 0; e < 8; ++e) for (int o = lpr; o < 64; o <<= 1) acc[e] += __shfl_xor(acc[e], o, 64);
        __syncthreads();                                                     // the previous flush has been read
        if (lane < lpr) {
#pragma unroll
            for (int e = 0; e < 8; ++e) if (e >= k.lo && e < k.hi) sh[(threadIdx.x >> 6) * 512 + k.cb + e] = acc[e];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < C; i += 256) put<D>(dst, i, (sh[i] + sh[512 + i]) + (sh[1024 + i] + sh[1536 + i]), as_d);
    }
}

template <typename TX, typename TB, bool GATE> struct BwdRow { Chunk<TX> dh, h; Chunk<TB> dy, b, g[1]; float keep; floatx4 st; };

// Waves a SIMD, which bounds the registers (512 / waves); the grid is what is resident then: a second, partial round of workgroups would
// run at a fraction of the waves (MiT stage 1: 1024 workgroups 203 us, 768 169 us)
__host__ __device__ constexpr int bwd_waves(bool narrow, bool post, int gate) { return narrow ? (!post && gate == 0 ? 4 : 3) : post ? 2 : 3; }

template <typename TX, typename TB, int WAVES, bool POST, int GATE>
__global__ __launch_bounds__(WAVES > 1 ? WAVES * 64 : 256, WAVES > 4 ? 2 : bwd_waves(sizeof(TX) == 2, POST, GATE)) void resnorm_bwd_kernel(ResnormBwdArgs a) {
    constexpr int THREADS = WAVES > 1 ? WAVES * 64 : 256;
    extern __shared__ __attribute__((aligned(16))) float vec[];              // post weight | post bias | scale | pre weight
    __shared__ float sh[WAVES > 1 ? 4 * WAVES : 4 * 512];
    int turn = 0;
    const int lpr = WAVES > 1 ? THREADS : a.lpr, lane = threadIdx.x & 63, lig = WAVES > 1 ? (int)threadIdx.x : lane & (lpr - 1), lanes = WAVES > 1 ? 64 : lpr;
    const int rpw = WAVES > 1 ? 1 : 64 / lpr;
    const int lr = WAVES > 1 ? 0 : lane / lpr, groups = WAVES > 1 ? 1 : 4 * rpw;   // this lane's row among the wave's; rows a workgroup takes at once
    const int wave_first = WAVES > 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * rpw;
    const Cols k = cols_of(lig * 8, a.C);
    const float invC = 1.f / a.C;
    const int vlen = lpr * 8;
    if (POST) { stage_vec(vec, a.post_w, 1.f, a.C, lpr, THREADS); stage_vec(vec + vlen, a.post_b, 0.f, a.C, lpr, THREADS); }
    stage_vec(vec + 2 * vlen, a.scale, 1.f, a.C, lpr, THREADS);
    if (a.pre) stage_vec(vec + 3 * vlen, a.pre_w, 1.f, a.C, lpr, THREADS);
    __syncthreads();
    auto sums = [&](const float (&g)[8], const float (&hat)[8], float& s1, float& s2) {      // a channel counts once
        if (a.ragged == 2) {
            const Cols own = here(k);
#pragma unroll
            for (int e = 0; e < 8; ++e) { const float v = e < own.lo || e >= own.hi ? 0.f : g[e]; s1 += v; s2 = fmaf(v, hat[e], s2); }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) { s1 += g[e]; s2 = fmaf(g[e], hat[e], s2); }
            if (a.ragged && lig * 8 >= a.C) { s1 = 0.f; s2 = 0.f; }
        }
    };
    float dwp[8] = {}, dbp[8] = {}, dwq[8] = {}, dbq[8] = {}, dsc[8] = {}, dgs[8] = {};
    for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        // a unit: every units_per_sample-th step of a sample's rows, so that the workgroups at work read one stretch of memory together
        // (a contiguous share each puts thousands of streams a power of two apart: MiT stage 1 210 -> 203 us)
        const int smp_u = unit / a.units_per_sample;
        const int begin = smp_u * a.sample_rows, end = begin + a.sample_rows;
        const int start = (unit - smp_u * a.units_per_sample) * groups, stride = a.units_per_sample * groups;
        Chunk<TB> unit_gate;
        if constexpr (GATE == 1) load_chunk(unit_gate, at<TB>(a.gate, smp_u, a.ldg, (unsigned)k.cb), a.C);
        // as the forward: two rows of registers, and the same number of steps for everybody who shares a row sum
        auto load = [&](BwdRow<TX, TB, GATE == 2>& t, int i) {
            const int row = begin + wave_first + i < end ? begin + wave_first + i : end - 1;   // the wave's first row
            const unsigned l = row + lr < end ? (unsigned)lr : 0u, cb = (unsigned)k.cb;
            t.keep = a.keep ? a.keep[GATE == 1 ? (unsigned)smp_u : fdiv((unsigned)row + l, a.per_sample)] : 1.f;
            load_chunk(t.dy, at<TB>(a.dy, row, a.lddy, l * (unsigned)a.lddy + cb), a.C);
            load_chunk(t.h, at<TX>(a.h, row, a.ldh, l * (unsigned)a.ldh + cb), a.C);
            load_chunk(t.dh, at<TX>(a.dh, row, a.lddh, l * (unsigned)a.lddh + cb), a.C);
            load_chunk(t.b, at<TB>(a.b, row, a.ldb, l * (unsigned)a.ldb + cb), a.C);
            if constexpr (GATE == 2) load_chunk(t.g[0], at<TB>(a.gate, row, a.ldg, l * (unsigned)a.ldg + cb), a.C);
            t.st = *at<floatx4>(a.stats, row, 1, l);
        };
        auto work = [&](BwdRow<TX, TB, GATE == 2>& t, int i) {
            const int row = begin + wave_first + i;
            const bool there = row + lr < end, ok = there && k.lo < k.hi;
            const unsigned dense = (unsigned)(lr * a.C + k.cb);
            if (row + rpw > end && !there) {                                 // a lane without a row adds nothing to the columns, infinities neither
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    t.dy.set(e, 0.f); t.dh.set(e, 0.f); t.h.set(e, 0.f); t.b.set(e, 0.f);
                    if constexpr (GATE == 2) t.g[0].set(e, 0.f);
                }
                t.st = floatx4{0.f, 0.f, 0.f, 0.f};
            }
                float d[8], hat[8], v[8];
                if (a.has_dh) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] = t.dh.get(e);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] = 0.f;
                }
                if (a.has_dy) {                                              // through the norm behind h
                    const float mh = t.st[2], rh = t.st[3];
                    float g[8], s1 = 0.f, s2 = 0.f;
                    vec_chunk(v, vec + 3 * vlen, lig, lpr);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float gy = t.dy.get(e);
                        hat[e] = (t.h.get(e) - mh) * rh;
                        dwp[e] = fmaf(gy, hat[e], dwp[e]); dbp[e] += gy;
                        g[e] = gy * v[e];
                    }
                    sums(g, hat, s1, s2);
                    row_sum2<WAVES>(s1, s2, lanes, sh, turn);
                    s1 = a.pre == 1 ? s1 * invC : 0.f; s2 *= invC;
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] = fmaf(rh, fmaf(-hat[e], s2, g[e] - s1), d[e]);
                }
                if (ok) {
                    Chunk<TX> o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o.set(e, d[e] * a.alpha);
                    store_chunk(o, at((TX*)a.dx, row, a.C, dense), a.C);
                }
                // dn, the scale's and the gate's gradients; n = hat w + bias
                float act[8], nn[8];
                const float mu = t.st[0], r = t.st[1];
                if (a.keep) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] *= t.keep;
                }
                if constexpr (POST) {
                    float w[8];
                    vec_chunk(w, vec, lig, lpr); vec_chunk(v, vec + vlen, lig, lpr);
#pragma unroll
                    for (int e = 0; e < 8; ++e) { hat[e] = (t.b.get(e) - mu) * r; nn[e] = fmaf(hat[e], w[e], v[e]); }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) nn[e] = t.b.get(e);
                }
                vec_chunk(v, vec + 2 * vlen, lig, lpr);
#pragma unroll
                for (int e = 0; e < 8; ++e) nn[e] *= d[e];
                if constexpr (GATE != 0) {
                    const Chunk<TB>& g = GATE == 1 ? unit_gate : t.g[0];
                    if (a.act) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) act[e] = sigmoid_f(g.get(e));
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) act[e] = g.get(e);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) { dsc[e] = fmaf(nn[e], act[e], dsc[e]); d[e] *= v[e] * act[e]; nn[e] *= v[e]; }
                    if (a.act) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) nn[e] *= fmaf(-act[e], act[e], act[e]);
                    }
                    if constexpr (GATE == 1) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) dgs[e] += nn[e];
                    } else if (ok) {
                        Chunk<TB> o;
#pragma unroll
                        for (int e = 0; e < 8; ++e) o.set(e, nn[e]);
                        store_chunk(o, at((TB*)a.dgate, row, a.C, dense), a.C);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) { dsc[e] += nn[e]; d[e] *= v[e]; }
                }
                if constexpr (POST) {                                        // through the norm of b
                    float s1 = 0.f, s2 = 0.f;
                    vec_chunk(v, vec, lig, lpr);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        dwq[e] = fmaf(d[e], hat[e], dwq[e]); dbq[e] += d[e];
                        d[e] *= v[e];
                    }
                    sums(d, hat, s1, s2);
                    row_sum2<WAVES>(s1, s2, lanes, sh, turn);
                    s1 = a.post == 1 ? s1 * invC : 0.f; s2 *= invC;
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] = r * fmaf(-hat[e], s2, d[e] - s1);
                }
                if (ok) {
                    Chunk<TB> o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o.set(e, d[e]);
                    store_chunk(o, at((TB*)a.db, row, a.C, dense), a.C);
                }
        };
        BwdRow<TX, TB, GATE == 2> r0, r1;
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
            for (int e = 0; e < 8; ++e) dgs[e] = 0.f;
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

// Joins the partial sums in a fixed order: workgroup row blockIdx.x < slots is a vector's gradient, the others are samples' gates.
// 32 columns x 32 parts a workgroup, four columns a thread: whole 128-byte lines, eight of them in flight a thread (2048 columns of three
// vectors from 1024 workgroups, 25 MB: 15.6 us with eight columns a workgroup, 6.1 us now).
template <typename TB>
__global__ __launch_bounds__(256) void resnorm_join_kernel(const float* __restrict__ partial, int blocks, int slots, float* __restrict__ out,
        const float* __restrict__ gate_partial, int units_per_sample, TB* __restrict__ dgate, int C) {
    __shared__ float sh[32][33];
    const int cx = (threadIdx.x & 7) * 4, part = threadIdx.x >> 3, col = blockIdx.y * 32 + cx;
    const bool vec = (int)blockIdx.x < slots;
    const int smp = (int)blockIdx.x - slots;
    const float* p = (vec ? partial + (int64_t)blockIdx.x * C : gate_partial + (int64_t)smp * units_per_sample * C) + col;
    const int64_t step = vec ? (int64_t)slots * C : C;
    const int count = vec ? blocks : units_per_sample, n = C - col;
    floatx4 s = {0.f, 0.f, 0.f, 0.f};
    if (n >= 4) {
#pragma unroll 8
        for (int i = part; i < count; i += 32) s += ((const Fl4u*)(p + (int64_t)i * step))->v;
    } else if (n > 0) {
        for (int i = part; i < count; i += 32)
#pragma unroll
            for (int e = 0; e < 3; ++e) if (e < n) s[e] += p[(int64_t)i * step + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sh[part][cx + e] = s[e];
    __syncthreads();
    const int mine = blockIdx.y * 32 + (int)threadIdx.x;
    if (threadIdx.x < 32 && mine < C) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += sh[i][threadIdx.x];
        if (vec) out[(int64_t)blockIdx.x * C + mine] = t; else dgate[(int64_t)smp * C + mine] = from_f<TB>(t);
    }
}

// ---------------------------------------------------------------- C ABI
static int waves_of(int C) { return C <= 512 ? 1 : C <= 1024 ? 2 : C <= 2048 ? 4 : 8; }
static int lanes_of(int C) { int l = 1; while (l * 8 < C && l < 64) l <<= 1; return l; }

struct ResnormPlan { int waves, lpr, slots, blocks, units, units_per_sample; int64_t sample_rows; };
static ResnormPlan resnorm_plan(int64_t rows, int64_t rows_per_sample, int C, int post, int pre, int gate_mode, bool scale, bool narrow) {
    ResnormPlan p;
    p.waves = waves_of(C); p.lpr = lanes_of(C);
    p.slots = (pre ? 1 : 0) + (pre == 1 ? 1 : 0) + (post ? 1 : 0) + (post == 1 ? 1 : 0) + (scale ? 1 : 0);
    p.sample_rows = gate_mode == 1 ? rows_per_sample : rows;
    const int64_t samples = rows / p.sample_rows;
    const int simd = p.waves > 4 ? 2 : bwd_waves(narrow, post != 0, gate_mode);
    const int64_t most = 256 * 4 * simd / (p.waves > 1 ? p.waves : 4);       // workgroups
    const int64_t step = p.waves > 1 ? 1 : 4 * (64 / p.lpr);                 // rows a workgroup takes at once
    int64_t per = most / samples;                                            // units of a sample: enough for all workgroups, each of at least one step
    if (per > cdiv(p.sample_rows, step)) per = cdiv(p.sample_rows, step);
    if (per < 1) per = 1;
    p.units_per_sample = (int)per;
    const int64_t units = samples * p.units_per_sample;
    p.units = (int)units;
    p.blocks = (int)(units < most ? units : most);
    return p;
}

extern "C" int64_t ss_resnorm_bwd_workspace(int64_t rows, int64_t rows_per_sample, int C, int post, int pre, int gate_mode, int has_scale) {
    if (rows <= 0 || rows_per_sample <= 0 || C <= 0 || C > SS_RESNORM_MAX_C || rows >= SS_RESNORM_MAX_ROWS) return 0;
    if (gate_mode == 1 && rows_per_sample == 1) gate_mode = 2;
    int64_t most = 0;                                                        // over the types
    for (int narrow = 0; narrow < 2; ++narrow) {
        const ResnormPlan p = resnorm_plan(rows, rows_per_sample, C, post, pre, gate_mode, has_scale != 0, narrow != 0);
        const int64_t need = ((int64_t)p.blocks * p.slots + (gate_mode == 1 && p.units_per_sample > 1 ? p.units : 0)) * C * 4;
        if (need > most) most = need;
    }
    return most;
}

extern "C" int ss_resnorm_bwd(int x_dtype, int b_dtype, const void* dh, int64_t lddh, const void* dy, int64_t lddy, const void* h, int64_t ldh,
                              const void* b, int64_t ldb, const void* gate, int64_t ldg, int gate_mode, int act, const float* scale, const float* keep,
                              float alpha, int post, const float* post_w, const float* post_b, int pre, const float* pre_w, const float* stats, void* dx,
                              void* db, void* dgate, float* dvec, int64_t rows, int64_t rows_per_sample, int C, float* workspace, int64_t ws_bytes,
                              hipStream_t stream) {
    if (gate_mode == 1 && rows_per_sample == 1) gate_mode = 2;               // a sample of one row
    if (int rc = resnorm_check("ss_resnorm_bwd", x_dtype, b_dtype, rows, rows_per_sample, C, post, pre, gate_mode, act, gate, post_w, post_b, pre_w, nullptr, false)) return rc;
    SS_CHECK(b && stats && dx && db && (dh || dy) && (!dy || (pre && h)) && (!gate || dgate) && lddh >= 0 && lddy >= 0 && ldh >= 0 && ldb >= 0 && ldg >= 0 &&
             lddh < SS_RESNORM_MAX_LD && lddy < SS_RESNORM_MAX_LD && ldh < SS_RESNORM_MAX_LD && ldb < SS_RESNORM_MAX_LD && ldg < SS_RESNORM_MAX_LD,
             "ss_resnorm_bwd: bad arguments");
    const ResnormPlan p = resnorm_plan(rows, rows_per_sample, C, post, pre, gate_mode, scale != nullptr, x_dtype == SS_BF16);
    const int64_t need = ((int64_t)p.blocks * p.slots + (gate_mode == 1 && p.units_per_sample > 1 ? p.units : 0)) * C * 4;
    SS_CHECK((p.slots == 0 || dvec) && (need == 0 || (workspace && ws_bytes >= need)), "ss_resnorm_bwd: workspace too small (%lld of %lld bytes)",
             (long long)ws_bytes, (long long)need);
    ResnormBwdArgs a;
    a.has_dh = dh != nullptr; a.has_dy = dy != nullptr;
    if (!dh) { dh = h; lddh = ldh; }
    if (!dy) { dy = b; lddy = ldb; h = dh; ldh = lddh; }
    a.dh = dh; a.dy = dy; a.h = h; a.b = b; a.gate = gate; a.dx = dx; a.db = db; a.dgate = dgate; a.stats = stats; a.post_w = post_w; a.post_b = post_b;
    a.scale = scale; a.keep = keep; a.pre_w = pre_w; a.partial = workspace; a.gate_partial = gate_mode == 1 && p.units_per_sample > 1 ? workspace + (int64_t)p.blocks * p.slots * C : nullptr;
    a.lddh = (int)lddh; a.lddy = (int)lddy; a.ldh = (int)ldh; a.ldb = (int)ldb; a.ldg = (int)ldg; a.sample_rows = (int)p.sample_rows;
    a.per_sample = fast_div((unsigned)rows_per_sample); a.units = p.units; a.units_per_sample = p.units_per_sample; a.slots = p.slots;
    a.ragged = C % 8 ? 2 : C != (p.waves > 1 ? p.waves * 64 : p.lpr) * 8;
    a.C = C; a.lpr = p.lpr; a.post = post; a.pre = pre; a.gate_mode = gate_mode; a.act = act; a.alpha = alpha;
    const size_t shm = (size_t)4 * (p.waves > 1 ? p.waves * 64 : p.lpr) * 8 * sizeof(float);
#define SS_RN_L(TX, TB, W, P, G) hipLaunchKernelGGL((resnorm_bwd_kernel<TX, TB, W, P, G>), dim3((unsigned)p.blocks), dim3(W > 1 ? W * 64 : 256), shm, stream, a)
#define SS_RN_G(TX, TB, W, P) do { if (gate_mode == 0) SS_RN_L(TX, TB, W, P, 0); else if (gate_mode == 1) SS_RN_L(TX, TB, W, P, 1); \
        else SS_RN_L(TX, TB, W, P, 2); } while (0)
#define SS_RN_P(TX, TB, W) do { if (post) SS_RN_G(TX, TB, W, true); else SS_RN_G(TX, TB, W, false); } while (0)
#define SS_RN_W(TX, TB) do { switch (p.waves) { case 1: SS_RN_P(TX, TB, 1); break; case 2: SS_RN_P(TX, TB, 2); break; \
        case 4: SS_RN_P(TX, TB, 4); break; default: SS_RN_P(TX, TB, 8); } } while (0)
    if (x_dtype == SS_BF16) SS_RN_W(bf16, bf16); else if (b_dtype == SS_BF16) SS_RN_W(float, bf16); else SS_RN_W(float, float);
    SS_LAUNCH_CHECK();
    const int64_t join = p.slots + (a.gate_partial ? rows / rows_per_sample : 0);
    if (join > 0) {
        const dim3 grid((unsigned)join, (unsigned)cdiv(C, 32));
        if (b_dtype == SS_BF16) hipLaunchKernelGGL(resnorm_join_kernel<bf16>, grid, dim3(256), 0, stream, workspace, p.blocks, p.slots, dvec,
                                                   a.gate_partial, p.units_per_sample, (bf16*)dgate, C);
        else hipLaunchKernelGGL(resnorm_join_kernel<float>, grid, dim3(256), 0, stream, workspace, p.blocks, p.slots, dvec, a.gate_partial,
                                p.units_per_sample, (float*)dgate, C);
        SS_LAUNCH_CHECK();
    }
    return 0;
}
