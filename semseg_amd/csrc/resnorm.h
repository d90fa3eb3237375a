// What the forward and the backward of the residual update between two norms share: eight channels of a row, row sums, the vectors in LDS.
#pragma once
#include "common.h"

// ---------------------------------------------------------------- eight channels of a row
// Row starts need no alignment beyond the element's (odd widths, odd row strides): global memory takes the access as one.
struct __attribute__((packed, aligned(2))) Bf8u { bf16x8 v; };
struct __attribute__((packed, aligned(4))) Fl8u { floatx4 a, b; };
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
struct __attribute__((packed, aligned(2))) Bf6u { unsigned a, b, c; };
struct __attribute__((packed, aligned(4))) Fl6u { floatx4 a; floatx2 b; };
template <typename T, int E> struct Chunk;
template <> struct Chunk<bf16, 8> {
    bf16x8 v;
    __device__ __forceinline__ void load(const bf16* p) { v = ((const Bf8u*)p)->v; }
    __device__ __forceinline__ float get(int e) const { return (float)v[e]; }
    __device__ __forceinline__ void set(int e, float f) { v[e] = (bf16)f; }
    __device__ __forceinline__ void store(bf16* p) const { ((Bf8u*)p)->v = v; }
};
template <> struct Chunk<bf16, 6> {
    unsigned v[3];
    __device__ __forceinline__ void load(const bf16* p) { const Bf6u t = *(const Bf6u*)p; v[0] = t.a; v[1] = t.b; v[2] = t.c; }
    __device__ __forceinline__ float get(int e) const { return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16); }
    __device__ __forceinline__ void set(int e, float f) { bf16x2 t = __builtin_bit_cast(bf16x2, v[e >> 1]); t[e & 1] = (bf16)f; v[e >> 1] = __builtin_bit_cast(unsigned, t); }
    __device__ __forceinline__ void store(bf16* p) const { *(Bf6u*)p = Bf6u{v[0], v[1], v[2]}; }
};
template <> struct Chunk<float, 6> {
    floatx4 a;
    floatx2 b;
    __device__ __forceinline__ void load(const float* p) { a = ((const Fl6u*)p)->a; b = ((const Fl6u*)p)->b; }
    __device__ __forceinline__ float get(int e) const { return e < 4 ? a[e & 3] : b[e & 1]; }
    __device__ __forceinline__ void set(int e, float f) { if (e < 4) a[e & 3] = f; else b[e & 1] = f; }
    __device__ __forceinline__ void store(float* p) const { ((Fl6u*)p)->a = a; ((Fl6u*)p)->b = b; }
};
template <> struct Chunk<float, 8> {
    floatx4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = ((const Fl8u*)p)->a; b = ((const Fl8u*)p)->b; }
    __device__ __forceinline__ float get(int e) const { return e < 4 ? a[e & 3] : b[e & 3]; }
    __device__ __forceinline__ void set(int e, float f) { if (e < 4) a[e & 3] = f; else b[e & 3] = f; }
    __device__ __forceinline__ void store(float* p) const { ((Fl8u*)p)->a = a; ((Fl8u*)p)->b = b; }
};
template <typename T> struct Chunk<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ float get(int) const { return to_f(v); }
    __device__ __forceinline__ void set(int, float f) { v = from_f<T>(f); }
    __device__ __forceinline__ void store(T* p) const { *p = v; }
};
// The E channels of a lane: eight, six where that leaves fewer lanes idle, one in rows of less than eight, so that C >= E always.  They are
// [cb, cb + E), of which those from lo on count as its own.  At the end of a row whose width is no multiple of E the last chunk is moved
// back to end with the row, and a lane past the row's end reads that chunk too and owns nothing (lo = E): every load is a whole chunk
// inside the row, WITHOUT A BRANCH, not even one that the whole launch takes alike: behind a branch the compiler cannot count the loads
// in flight, a wait for one row's loads becomes a wait for all, and the next row's are not on their way any more (bf16, LN + LN +
// gate, 24 M elements, backward: C = 500 73 -> 65 us, 4096 100 -> 82; forward 500 50 -> 44, 4096 44 -> 40).  What two lanes
// hold of the same channel is the same to the last bit, so the moved chunk is stored whole as well; only sums count a channel once.
struct Cols { int cb, lo; };
template <int E> __device__ __forceinline__ Cols cols_of(int c, int C) {
    const int n = C - c;
    Cols r;
    r.cb = n >= E ? c : C - E;
    r.lo = n >= E ? 0 : n <= 0 ? E : E - n;
    return r;
}
// compared where it is used: sixteen lane masks kept over a loop do not fit the scalar registers
__device__ __forceinline__ Cols here(Cols k) { asm volatile("" : "+v"(k.lo)); return k; }

// Address of a lane's element: a row that the whole wave agrees on (64 bits, scalar registers) and the lane's offset from it (32 bits): one
// vector register a tensor instead of two for every pointer.  The host keeps 64 row strides below 2^32 bytes.
template <typename T> __device__ __forceinline__ T* at(T* base, int row, int ld, unsigned off) {
    return (T*)((char*)(base + (int64_t)row * ld) + off * (unsigned)sizeof(T));
}
template <typename T> __device__ __forceinline__ const T* at(const void* base, int row, int ld, unsigned off) {
    return (const T*)((const char*)((const T*)base + (int64_t)row * ld) + off * (unsigned)sizeof(T));
}
#define SS_RESNORM_MAX_LD (1LL << 23)
#define SS_RESNORM_MAX_ROWS (1LL << 30)

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
    if constexpr (WAVES == 1) __builtin_amdgcn_sched_barrier(0);            // what follows is not moved up here: it would only take registers
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
template <int WAVES> __device__ __forceinline__ void row_stats(double s, double q, int kind, double inv_c, double eps, int lanes, double* sh, int& turn, float& mu, float& r) {
    row_sum2<WAVES>(s, q, lanes, sh, turn);
    const double m = kind == 1 ? s * inv_c : 0.0;
    double var = fma(-m, m, q * inv_c);
    var = var > 0.0 ? var : (var < 0.0 ? 0.0 : var);                        // NaN stays
    mu = (float)m; r = (float)rsqrt_d(var + eps);
}
__device__ __forceinline__ float sigmoid_f(float v) { return __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

// ---------------------------------------------------------------- the vectors (weights, biases, scale) in LDS
// One row of `chunks` chunks per vector, the first four and the other channels of a chunk apart: lanes read 16 bytes each, 16 bytes apart,
// then 16 or 8.
template <int E> __device__ __forceinline__ void put_chunk(float* sh, const float (&v)[E], int chunk, int chunks) {
    if constexpr (E == 1) sh[chunk] = v[0];
    else {
        *(floatx4*)(sh + chunk * 4) = floatx4{v[0], v[1], v[2], v[3]};
        if constexpr (E == 8) *(floatx4*)(sh + chunks * 4 + chunk * 4) = floatx4{v[4], v[5], v[6], v[7]};
        else *(floatx2*)(sh + chunks * 4 + chunk * 2) = floatx2{v[4], v[5]};
    }
}
// a lane's chunk of a vector, or the value that stands for one that is not given
template <int E> __device__ __forceinline__ void load_vec(float (&v)[E], const float* p, float otherwise, const Cols& k) {
    Chunk<float, E> t;
    if (p) t.load(p + k.cb);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = p ? t.get(e) : otherwise;
}
template <int E> __device__ __forceinline__ void vec_chunk(float (&v)[E], const float* sh, int chunk, int chunks) {
    if constexpr (E == 1) v[0] = sh[chunk];
    else {
        const floatx4 a = *(const floatx4*)(sh + chunk * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = a[e];
        if constexpr (E == 8) {
            const floatx4 b = *(const floatx4*)(sh + chunks * 4 + chunk * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 + e] = b[e];
        } else {
            const floatx2 b = *(const floatx2*)(sh + chunks * 4 + chunk * 2);
            v[4] = b[0]; v[5] = b[1];
        }
    }
}

// ---------------------------------------------------------------- C ABI: what both entries check
#define SS_RESNORM_MAX_C 4096
static inline int resnorm_check(const char* who, int x_dtype, int b_dtype, int64_t rows, int64_t rows_per_sample, int C, int post, int pre, int gate_mode,
                         int act, const void* gate, const float* post_w, const float* post_b, const float* pre_w, const float* pre_b, bool biases) {
    SS_CHECK((x_dtype == SS_F32 && (b_dtype == SS_F32 || b_dtype == SS_BF16)) || (x_dtype == SS_BF16 && b_dtype == SS_BF16),
             "%s: stream / branch types must be f32 / f32, bf16 / bf16 or f32 / bf16, got codes %d / %d", who, x_dtype, b_dtype);
    SS_CHECK(rows > 0 && rows < SS_RESNORM_MAX_ROWS && rows_per_sample > 0 && rows % rows_per_sample == 0, "%s: bad row counts (%lld, %lld a sample)", who,
             (long long)rows, (long long)rows_per_sample);
    SS_CHECK(C > 0 && C <= SS_RESNORM_MAX_C, "%s: C=%d must be 1 to %d", who, C, SS_RESNORM_MAX_C);
    SS_CHECK(post >= 0 && post <= 2 && pre >= 0 && pre <= 2 && gate_mode >= 0 && gate_mode <= 2 && act >= 0 && act <= 1, "%s: bad codes", who);
    SS_CHECK((gate_mode != 0) == (gate != nullptr), "%s: a gate and its layout go together", who);
    SS_CHECK((!post || post_w) && (!pre || pre_w), "%s: a norm needs its weight", who);
    SS_CHECK(!biases || ((post == 1 || !post_b) && (pre == 1 || !pre_b)), "%s: only LayerNorm takes a bias", who);
    return 0;
}

