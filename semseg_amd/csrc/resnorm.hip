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
// Work split: a row is a power of two of lanes with eight channels each, or six where that leaves fewer lanes idle.  Up to 512 channels a
// wave holds 64 / lanes rows; above, the WAVES of a workgroup share the row and join their sums through LDS.  Row sums are taken in double, sum and sum of squares in ONE pass: the
// variance does not cancel (double holds the square of any float exactly), one reduction serves mean and variance, and the result is
// the same to the last bit of a float whatever the split -- h is rounded to 8 bits behind it, and an h near the border of two values
// would otherwise depend on the order of a sum.  Products and sums up to h are rounded one by one (no contraction) for the same reason.
#include "resnorm_fwd.h"

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
    int waves = 1, nch = 1, width = C < 8 ? 1 : 8;
    const int chunks = (int)cdiv(C, width);
    // Lanes of a row, measured at 24 M elements:
    // - a stream in 32 bits is bound by its bytes: one chunk a lane, whole lines in a load (C = 96: 83 us, 96 in four lanes x 3; 320: 80 in 64
    //   lanes, 103 in sixteen x 3; 768 in two waves: 81, 97 in 32 lanes x 3, and in chunks of six 82);
    // - a bf16 stream with norms and gates is bound by vector instructions: up to 512 channels up to four chunks a lane so that the fewest lanes
    //   are idle, of those the most lanes (C = 96 in 4 x 3: 43 us, 51 in 16; 384 in 16 x 3: 44, 57 in 64; 128 in 16: 41, 43 in 8 x 2); above, the
    //   waves of a workgroup one chunk a lane, of six channels where they reach (768: 40 us, 47 in eights, 47 in one wave x 3; 1024: 38, 50 in
    //   one wave x 4; 1536: 42, 48 in eights);
    // - with rows too few for a wave on every SIMD, as many lanes as there are chunks (1 row of 512: 6.4 -> 5.0 us).
    if (chunks > 64) {
        waves = chunks <= 128 ? 2 : chunks <= 256 ? 4 : 8;
        a.lpr = waves * 64;
        if (x_dtype == SS_BF16 && cdiv(C, 6) <= a.lpr) width = 6;
    } else if (x_dtype == SS_F32 || rows * chunks < 64 * 1024 || width == 1) { a.lpr = 1; while (a.lpr < chunks) a.lpr <<= 1; }
    else {
        int slots = 1 << 30;
        for (int l = 64; l >= 1; l >>= 1) {
            const int n = (int)cdiv(chunks, l);
            if (n <= 4 && l * n < slots) { slots = l * n; a.lpr = l; nch = n; }
        }
    }
    a.ragged = C % width != 0 ? 2 : C != a.lpr * nch * width;
    const int64_t want = waves > 1 ? rows : cdiv(rows, 4 * (64 / a.lpr)), most = waves > 1 ? 4096 / waves : 1024;
    const ResnormFwdLaunch l{x_dtype, b_dtype, waves, nch, (int)(want < most ? want : most)};
    if (width == 6) resnorm_fwd_launch6(a, l, stream); else if (width == 1) resnorm_fwd_launch1(a, l, stream); else resnorm_fwd_launch<8>(a, l, stream);
    SS_LAUNCH_CHECK();
    return 0;
}
