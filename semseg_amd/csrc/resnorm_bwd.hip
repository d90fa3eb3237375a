// Backward of the residual update between two norms (resnorm_bwd.h: the kernel): its geometry, the join of its partial sums, the entries.
#include "resnorm_bwd.h"

struct __attribute__((packed, aligned(4))) Fl4u { floatx4 v; };

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
static int lanes_of(int C) { int l = 1; const int chunks = C < 8 ? C : (int)cdiv(C, 8); while (l < chunks && l < 64) l <<= 1; return l; }
// Six channels a lane instead of eight where the same lanes reach: a quarter less work for every lane and fewer registers, nothing idle at
// 3 x 2^k (24 M elements, TB/s: LN + LN + gate in bf16, C = 384 3.7 -> 4.8, 96 3.9 -> 4.7, 320 3.3 -> 4.2, 768 3.3 -> 3.9; RMS twice in f32,
// 384 4.2 -> 4.8)
static int width_of(int C, int lanes) { return C < 8 ? 1 : C > 8 && cdiv(C, 6) <= lanes ? 6 : 8; }

struct ResnormPlan { int waves, lpr, width, slots, blocks, units, units_per_sample; int64_t sample_rows; };
static ResnormPlan resnorm_plan(int64_t rows, int64_t rows_per_sample, int C, int post, int pre, int gate_mode, bool scale, bool narrow) {
    ResnormPlan p;
    p.waves = waves_of(C); p.lpr = lanes_of(C);
    p.width = width_of(C, p.waves > 1 ? p.waves * 64 : p.lpr);
    p.slots = (pre ? 1 : 0) + (pre == 1 ? 1 : 0) + (post ? 1 : 0) + (post == 1 ? 1 : 0) + (scale ? 1 : 0);
    p.sample_rows = gate_mode == 1 ? rows_per_sample : rows;
    const int64_t samples = rows / p.sample_rows;
    const int simd = bwd_waves(p.width, p.waves, narrow, post != 0, gate_mode);
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
    a.ragged = C % p.width ? 2 : C != (p.waves > 1 ? p.waves * 64 : p.lpr) * p.width;
    a.C = C; a.lpr = p.lpr; a.post = post; a.pre = pre; a.gate_mode = gate_mode; a.act = act; a.alpha = alpha;
    const ResnormLaunch l{x_dtype, b_dtype, p.waves, p.lpr, p.blocks};
    if (p.width == 6) resnorm_bwd_launch6(a, l, stream); else if (p.width == 1) resnorm_bwd_launch1(a, l, stream); else resnorm_bwd_launch<8>(a, l, stream);
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
