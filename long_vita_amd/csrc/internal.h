// Internal launch interfaces between the translation units of liblvattn.
#pragma once
#include "common.h"

// Rules that change a score before the softmax.  A kernel instantiated with MOD != 0 works on t = log2(e) * score, where
//   score = cap * tanh(scale * q.k / cap)   (LV_SCORE_CAP; else scale * q.k)
//           - slope[head] * |query position - key position|   (LV_SCORE_BIAS)
// and always honours the descriptor's prefix (word 7).  With x = 2 log2(e) scale q.k / cap,
//   cap tanh = cap (1 - 2 / (2^x + 1)):  one exponential and one reciprocal, exact limits on both sides (2^x = inf gives cap,
// 0 gives -cap).  The two terms nearly cancel where the score is small beside the cap: the absolute error is about 1.4e-7 cap,
// 9e-6 at a cap of 64, 1e-3 at 1e4.  Caps above LV_SCORE_WIDE_CAP (LV_SCORE_WIDE) therefore take, for |x| < log2(e) (scores under
// half the cap),
//   cap tanh = score (1 + x^2 (a1 + x^2 (a2 + x^2 (a3 + x^2 a4)))),
// a polynomial fitted to tanh(y) / y for |y| <= 1/2 (least squares, weights moved until the error is level: 1.4e-8); with either
// form the error is then below 4e-7 of the score itself, whatever the cap.  That costs about ten vector instructions per score,
// so caps that models train with (20 to 50) do not take it: 8,192 packed rows, 40 / 8 heads, cap 50 / 65, forward 351 / 640 us, training
// 1,403 / 2,138 us.  The wide kernels always hold the bias (slopes may be null: 0), so that one more variant serves both.
#define LV_SCORE_CAP 1
#define LV_SCORE_BIAS 2
#define LV_SCORE_RULE 4        // set in every MOD: prefix rows, no other rule needed
#define LV_SCORE_WIDE 8        // with CAP and BIAS
#define LV_SCORE_WIDE_CAP 64.f
#define LV_SCORE_BITS(mod) ((mod) & (LV_SCORE_CAP | LV_SCORE_BIAS | LV_SCORE_WIDE))
struct ScoreRule {
    float cap_in;              // 2 log2(e) scale / cap: the exponent of the tanh from the raw product q.k
    float cap_out;             // cap log2(e)
    float plus0;               // lv_score_plus: cap_out with a cap up to LV_SCORE_WIDE_CAP, else 0
    const float* slopes;       // [hq], device
};
#ifdef __HIPCC__
// -log2(e) slope of a head (MOD has LV_SCORE_BIAS)
template <int MOD>
__device__ __forceinline__ float lv_slope2(const ScoreRule& u, int head) {
    if constexpr (MOD & LV_SCORE_WIDE) if (!u.slopes) return 0.f;
    return -1.4426950408889634f * u.slopes[head];
}
// log2(e) cap tanh(x ln(2) / 2) of a wide cap; rc = 1 / (2^x + 1), c = scale log2(e)
__device__ __forceinline__ float lv_score_wide(float s, float c, float x, float rc, const ScoreRule& u) {
    const float z = x * x, near = s * c;
    float a = __builtin_fmaf(z, 3.5919336e-06f, -9.193529e-05f);
    a = __builtin_fmaf(z, a, 0.001922566f);
    a = __builtin_fmaf(z, a, -0.040037528f);
    return __builtin_fabsf(x) < 1.4426950f ? __builtin_fmaf(near, z * a, near) : __builtin_fmaf(-2.f * u.cap_out, rc, u.cap_out);
}
// raw product s -> t; `dist` = signed distance of the two positions
template <int MOD>
__device__ __forceinline__ float lv_score(float s, float c, const ScoreRule& u, float nslope2, float dist) {
    float t;
    if constexpr (MOD & LV_SCORE_WIDE) {
        const float x = s * u.cap_in;
        t = lv_score_wide(s, c, x, __builtin_amdgcn_rcpf(fast_exp2(x) + 1.f), u);
    } else if constexpr (MOD & LV_SCORE_CAP) t = __builtin_fmaf(-2.f * u.cap_out, __builtin_amdgcn_rcpf(fast_exp2(s * u.cap_in) + 1.f), u.cap_out);
    else t = s * c;
    if constexpr (MOD & LV_SCORE_BIAS) t = __builtin_fmaf(nslope2, __builtin_fabsf(dist), t);
    return t;
}
// t + (plus - lv_score_plus0): with a cap (not a wide one, beside which the constant's other terms would be lost) the caller's
// constant holds cap_out, so that no instruction per score adds it.
// quarter: a fourth of the tanh's derivative, 1 - tanh^2 = 1 - (1 - 2 rc)^2 = 4 (rc - rc^2); the 4 goes into the caller's last
// factor.  (Packed segments, 40 / 8 heads, cap 50: dQ 584 -> 577 us, dK / dV 700 -> 678 us.)
template <int MOD>
__device__ __forceinline__ float lv_score_plus0(const ScoreRule& u) { return (MOD & LV_SCORE_CAP) ? u.plus0 : 0.f; }
template <int MOD>
__device__ __forceinline__ float lv_score_plus(float s, float c, const ScoreRule& u, float nslope2, float dist, float plus, float* quarter = nullptr) {
    float t;
    if constexpr (MOD & LV_SCORE_CAP) {
        const float x = s * u.cap_in, rc = __builtin_amdgcn_rcpf(fast_exp2(x) + 1.f);
        if constexpr (MOD & LV_SCORE_WIDE) t = lv_score_wide(s, c, x, rc, u) + plus;
        else t = __builtin_fmaf(-2.f * u.cap_out, rc, plus);
        if (quarter) *quarter = __builtin_fmaf(-rc, rc, rc);
    } else {
        t = __builtin_fmaf(s, c, plus);
    }
    if constexpr (MOD & LV_SCORE_BIAS) t = __builtin_fmaf(nslope2, __builtin_fabsf(dist), t);
    return t;
}
#endif

struct FwdParams {
    const __bf16* q;
    const __bf16* k;
    const __bf16* v;
    __bf16* o;
    float* lse;
    const AttnDesc* desc;
    int n_blocks, hq, hkv, group;  // group = hq / hkv
    int q_rows_total, k_rows_total;
    int64_t q_rs, q_hs, k_rs, k_hs, v_rs, v_hs, o_rs, o_hs, lse_stride;
    float scale, scale_log2e;
    int head_per_xcd;   // workgroup order: every work item of a KV head on ONE XCD, back to back (set by the launchers)
    // rotary embedding applied to the query fragments as they are loaded (null = off): bf16 tables [tab_rows][d],
    // table row of tensor row i = pos[i] or i / tab_div; q_rot (optional) receives the rotated queries
    const __bf16* rope_cos;
    const __bf16* rope_sin;
    const int32_t* rope_pos;
    int64_t rope_tab_rows;
    int rope_tab_div;
    __bf16* q_rot;
    int64_t qr_rs, qr_hs;
    ScoreRule score;    // read by the MOD != 0 kernels only, as are the two below
    float* o_f32;       // not null: results go here, unrounded, [rows][hq][d] contiguous, instead of o
    uint8_t* o_lo;      // not null: what the rounding of o cut off, [rows][hq][d] contiguous (lv_low_byte)
};
// An fp32 number as its bf16 rounding plus one byte: the eight bits below the bf16 mantissa, before the rounding.  The tie that
// rounds down would read like one that rounds up; it is stored a step lower.  lv_join_low gives back 16 bits of mantissa.
#ifdef __HIPCC__
__device__ __forceinline__ uint32_t lv_low_byte(float x) {
    const uint32_t u = __float_as_uint(x), b = (u >> 8) & 0xffu;
    return b - ((u & 0x1ffffu) == 0x8000u ? 1u : 0u);
}
__device__ __forceinline__ float lv_join_low(uint32_t bf16_bits, uint32_t b) {
    return __uint_as_float(((bf16_bits - (b >> 7)) << 16) | (b << 8) | 0x80u);
}
#endif
// Workgroup i of a launch runs on XCD i % 8, and every XCD has its own L2.  When ALL the work items of one KV head
// (query blocks x the group's query heads) fit on an XCD's 32 CUs at once, they are given consecutive slots of one XCD:
// the head's K / V then come into that L2 once instead of once per XCD that hosts one of its items (the vision
// tower: 1024 heads x 4-5 query blocks, where the plain order fetched K / V four times, L2 hit rate 41 %).
inline bool lv_head_per_xcd(const FwdParams& p) { return (int64_t)p.n_blocks * p.group <= 32 && p.hkv >= 8; }
#ifdef __HIPCC__
// Work item `blk` of a forward launch: the caller's descriptor, or (desc == nullptr: ONE dense segment, no descriptor
// memory at all) rows [blk * bm, + bm) of q_rows_total query rows against all k_rows_total keys; the causal rule is
// aligned to the END of both ranges (query row i sees keys j <= i + k_rows_total - q_rows_total).  Causal blocks are
// numbered from the last one down: heaviest first, as the host block builders order theirs.
__device__ __forceinline__ AttnDesc lv_fwd_desc(const FwdParams& p, int blk, int bm, bool causal) {
    if (p.desc) return p.desc[blk];
    if (causal) blk = p.n_blocks - 1 - blk;
    AttnDesc d;
    d.a_row0 = blk * bm;
    d.a_rows = min(bm, p.q_rows_total - d.a_row0);
    d.b_row0 = 0;
    d.out_delta = 0;
    d.band_p1 = 0;
    d.shift = causal ? p.k_rows_total - p.q_rows_total + d.a_row0 : 0;
    d.b_len = causal ? max(0, min(p.k_rows_total, d.a_rows + d.shift)) : p.k_rows_total;
    return d;
}
#endif
int lv_launch_fwd(const FwdParams& p, int d, int causal, int waves, hipStream_t stream);
int lv_launch_fwd_pp(const FwdParams& p, int d, int causal, hipStream_t stream);  // ping-pong form, 256-row items
int lv_launch_fwd_pp_score(const FwdParams& p, int d, int mod, hipStream_t stream);  // the same with p.score applied
int lv_launch_fwd_pp16(const FwdParams& p, int causal, hipStream_t stream);      // ping-pong form on 16x16x32 MFMAs, d = 128
int lv_launch_fwd_a4(const FwdParams& p, int causal, hipStream_t stream);        // one wave per SIMD, 64 query rows per wave, d = 128

// Incremental attention over a KV cache: q [batch, hq, d], k/v [batch, k_len, hkv, d], out [batch, hq, d].
#define LV_DECODE_MAX_SPLITS 256
#define LV_DECODE_TILE 128
#define LV_DECODE_SCRATCH_BYTES (8 << 20)   // partial results of lvattn_decode_noalloc, held by every GPU the library runs on
#define LV_MAX_DEVICES 64
struct DecodeParams {
    const __bf16* q;
    const __bf16* k;
    const __bf16* v;
    __bf16* o;
    float* lse;        // [batch, hq] or null
    float* part_o;     // [batch*hkv][n_split][group][d]
    float* part_lse;   // [batch*hkv][n_split][group]
    int batch, hq, hkv, group, k_len, chunk, n_split;
    int64_t q_bs, q_hs, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs, o_bs, o_hs;
    float scale, scale_log2e;
};
int lv_launch_decode(const DecodeParams& p, int d, hipStream_t stream);

// Drafted tokens over a KV cache: q [batch, n, hq, d], k / v [batch, rows, hkv, d], out [batch, n, hq, d].
#define LV_TREE_MAX_TOKENS 256
#define LV_TREE_MAX_BATCH 512
#define LV_TREE_MAX_SHARES 256
struct TreeParams {
    const __bf16* q;
    const __bf16* k;
    const __bf16* v;
    __bf16* o;
    float* lse;                  // [batch, n, hq] or null
    const int32_t* cache_lens;   // [batch]
    const int32_t* parents;      // [n] per sequence, or null: a chain
    int64_t parents_bs;
    float* part_o;               // [hkv][n_rb][slots][32 * WR][d]
    float* part_lse;             // the same without d
    int batch, n, rows, hq, hkv, group, n_rb, shares, slots, direct;
    int64_t q_bs, q_ns, q_hs, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs, o_bs, o_ns, o_hs;
    float scale, scale_log2e;
    ScoreRule score;
};
struct AcceptParams {
    __bf16* k;
    __bf16* v;
    float* weight;               // [batch, hkv, rows] or null
    const int32_t* cache_lens;
    const int32_t* path;         // [batch, n] ascending token numbers
    const int32_t* n_accept;     // [batch]
    int32_t* new_lens;           // [batch] or null
    int n, rows, hkv, d;
    int64_t k_bs, k_rs, k_hs, v_bs, v_rs, v_hs, w_bs, w_hs;
};

struct WeightParams {
    const __bf16* q;
    const __bf16* k;
    const float* lse;            // [batch, n, hq]
    const float* row_weight;     // [batch, n] or null: 1
    const float* w_in;           // [batch, hkv, rows]
    float* w_out;                // the same, may be w_in
    const int32_t* cache_lens;
    const int32_t* parents;
    int64_t parents_bs;
    float* row_const;            // [batch * hkv][3][rows_pad]
    float* part;                 // [pieces][batch * hkv][rows]
    uint32_t* dead;              // [batch * hkv][rows_pad / 256]: a row of these 256 counts for nothing
    int batch, n, rows, hq, hkv, group, pieces, shares, rows_pad, row0, rest;
    int64_t q_bs, q_ns, q_hs, k_bs, k_rs, k_hs, wi_bs, wi_hs, wo_bs, wo_hs;
    float scale_log2e;
    ScoreRule score;
};
struct EvictParams {
    const __bf16* k_in;
    const __bf16* v_in;
    const float* w_in;
    __bf16* k_out;
    __bf16* v_out;
    float* w_out;
    const int32_t* cache_lens;
    int32_t* index;              // [batch * hkv][keep]
    int32_t* new_lens;
    uint32_t* hist;              // [3][batch * hkv][2048]
    uint32_t* counts;            // [batch * hkv][chunks][2]
    uint32_t* thr;               // [batch * hkv][2]
    int batch, rows, hkv, keep, sink, recent, chunks, zero_fill;
    int64_t ki_bs, ki_rs, ki_hs, vi_bs, vi_rs, vi_hs, wi_bs, wi_hs, ko_bs, ko_rs, ko_hs, vo_bs, vo_rs, vo_hs, wo_bs, wo_hs;
};

#define LV_BWD_BLOCK_N_INTERNAL 128

struct BwdParams {
    const __bf16* q;
    const __bf16* k;
    const __bf16* v;
    const __bf16* dout;
    const float* lse;
    const float* delta;
    void* dq;    // bf16 (stored) or fp32 (accumulated), as dk / dv
    void* dk;
    void* dv;
    const AttnDesc* desc;    // key blocks (dK/dV kernel)
    const AttnDesc* qdesc;   // query blocks (dQ kernel)
    int n_blocks, n_qblocks, hq, hkv, group;
    int q_rows_total, k_rows_total;
    int64_t q_rs, q_hs, k_rs, k_hs, v_rs, v_hs, do_rs, do_hs, dq_rs, dq_hs, dk_rs, dk_hs, dv_rs, dv_hs, lse_stride;
    float scale, scale_log2e;
    int f32_store;   // fp32 results are stored, not added to what the buffers hold (accum_f32 == 2)
    ScoreRule score; // read by the MOD != 0 kernels only
};
int lv_launch_bwd(const BwdParams& p, int d, int causal, int accum, hipStream_t stream);
int lv_launch_bwd_dkdv_rs(const BwdParams& p, int d, int causal, int accum, hipStream_t stream);  // role-split dK/dV kernel
int lv_launch_bwd_dkdv_g(const BwdParams& p, int causal, int accum, hipStream_t stream);          // one wave per SIMD, gap-scheduled dK/dV kernel, d = 128
int lv_launch_bwd_dq_pp(const BwdParams& p, int d, int causal, int accum, hipStream_t stream);  // ping-pong dQ kernel
int lv_launch_bwd_dq_pp_score(const BwdParams& p, int d, int accum, int mod, hipStream_t stream);    // with p.score applied
int lv_launch_bwd_dkdv_rs_score(const BwdParams& p, int d, int accum, int mod, hipStream_t stream);
ScoreRule lv_score_rule(float scale, float softcap, const float* slopes);
int lv_score_mod(float softcap, const float* slopes);      // LV_SCORE_* bits of a rule
// error text of the calling thread (lvattn_last_error); returns `code`
int lv_fail(int code, const char* fmt, ...);
int lv_check_qkv(const void* q, const void* k, const void* v, int hq, int hkv, int d, int64_t q_rs, int64_t q_hs, int64_t k_rs,
                 int64_t k_hs, int64_t v_rs, int64_t v_hs);
// piece length that a simulated schedule of `copies` copies of these sweeps likes best on n_cu compute units; 0 = leave them whole
int lv_plan_sweeps(const int* sweep, int n, int copies, int n_cu, int fixed, int min_piece);
void lv_select_bwd_kernels(int dq, int dkdv);   // 0 default, 1 the earlier kernel, (dkdv) 2 the gap-scheduled kernel, < 0 unchanged
void lv_select_rs_units(int n);                  // 32-row units per iteration of the role-split dK/dV kernel: 1 or 2
int lv_launch_bwd_delta(const void* o, const void* dout, float* delta, int rows, int hq, int d, int64_t o_rs, int64_t o_hs,
                        int64_t do_rs, int64_t do_hs, int64_t lse_stride, hipStream_t stream);
int lv_launch_rope(const void* x, void* out, const void* cos_tab, const void* sin_tab, const int32_t* pos_ids, int64_t rows,
                   int heads, int d, int rot, int64_t x_rs, int64_t x_hs, int64_t o_rs, int64_t o_hs, int64_t tab_rows, int tab_div,
                   int conj, hipStream_t stream);
int lv_launch_rope_pack_kv(const void* k, const void* v, void* kv, const void* cos_tab, const void* sin_tab, const int32_t* pos_ids,
                           int64_t rows, int heads, int d, int rot, int64_t k_rs, int64_t k_hs, int64_t v_rs, int64_t v_hs,
                           int64_t tab_rows, int tab_div, hipStream_t stream);
int lv_launch_layernorm(const void* x, void* y, const void* gamma, const void* beta, int64_t rows, int h, int64_t x_rs,
                        int64_t y_rs, float eps, hipStream_t stream);
int lv_launch_bias_gelu(const void* x, const void* bias, void* y, int64_t rows, int h, hipStream_t stream);
int lv_launch_bias_gelu_bwd(const void* x, const void* bias, const void* dy, void* dx, int64_t rows, int h, hipStream_t stream);
int lv_layernorm_bwd_parts(int64_t rows);
int lv_launch_layernorm_bwd(const void* x, const void* dy, const void* gamma, void* dx, float* dgamma_dbeta, float* part,
                            int64_t rows, int h, int64_t x_rs, int64_t dy_rs, int64_t dx_rs, float eps, hipStream_t stream);
int lv_launch_bias_scale_residual(const void* x, const void* bias, const void* ls, const void* res, void* out, int64_t rows, int h,
                                  hipStream_t stream);
int lv_launch_bsr_layernorm(const void* x, const void* bias, const void* ls, const void* res, void* x1, void* y, const void* gamma,
                            const void* beta, int64_t rows, int h, float eps, hipStream_t stream);
int lv_launch_patchify(const void* img, void* out, int n, int c, int H, int W, int p, int kpad, hipStream_t stream);
int lv_launch_embed_tokens(const void* proj, const void* conv_bias, const void* cls, const void* pos, void* out, int n, int np,
                           int ncls, int h, hipStream_t stream);
