// Attention whose scores follow a rule of their own: a tanh cap, a bias that grows with distance, a prefix that every row of
// its segment sees.  Forward and backward, packed segments.
//
//   s_ij = scale q_i.k_j;  u_ij = cap tanh(s_ij / cap) (or s_ij);  t_ij = u_ij - slope_h |i - j|
//   visible: same segment and (j <= i or j < prefix) and (no band or j >= i - band)
//   O_i = sum_j softmax_j(t_ij) v_j,  lse_i = log sum_j exp t_ij
//   dT = P (dP - delta);  dS = dT (1 - tanh^2);  dQ = scale dS K;  dK = scale dS^T Q;  dV = P^T dO
//
// The products are those of plain attention, so the kernels are the ping-pong forward, the ping-pong dQ and the role-split
// dK/dV kernels instantiated with the rule applied to every raw product in their vector phase (lv_score in internal.h).  What
// the rule needs is not the matrix pipe: a cap adds an exponential and a reciprocal to the one exponential of the softmax.
// Measured, 40 / 8 heads of 128, forward / dQ / dK and dV within a training step: 8,192 packed rows with a cap 420 / 524 / 658 us,
// 12,288 rows with slopes 1,705 / 2,077 / 3,441 us.  With the cap the matrix pipe is busy 27 / 33 / 32 % of the cycles and vector
// instructions issue in 43 / 38 / 43 % of them: neither is full, the chain exponential - reciprocal - exponential of a tile is waited
// for.  With slopes 43 / 57 / 42 % and 39 / 48 / 41 %.
// This file holds the host side: work-item tables that know the prefix and the band (whole sweeps or sweeps cut into
// pieces), the choice of the piece length, and the entry points.
#include "internal.h"
#include "../../include/lvattn.h"

#include <algorithm>
#include <cstring>
#include <exception>
#include <vector>

namespace {

constexpr int kFwdRows = 256;
constexpr int kBwdKeys = LV_BWD_BLOCK_N_INTERNAL;

// a: the rows a work item owns, b: the range it sweeps; shift / prefix relative to the first swept (forward) or owned
// (backward) key: key j visible to row i iff j <= i + shift or j < prefix
struct Sweep { int a0, an, b0, bn, shift, prefix, band_p1; };

void sweeps_of(const int32_t* cu, int n_seg, int causal, int band, const int32_t* prefix, bool backward, std::vector<Sweep>& out) {
    for (int s = 0; s < n_seg; ++s) {
        const int base = cu[s], len = cu[s + 1] - cu[s];
        // without the causal rule every key is a prefix key
        const int pre = !causal ? len : (prefix ? std::min(prefix[s], len) : 0);
        const int band_p1 = band >= 0 ? band + 1 : 0;
        if (!backward) {
            for (int m = 0; m < len; m += kFwdRows) {
                const int rows = std::min(kFwdRows, len - m);
                const int first = band >= 0 ? std::max(0, m - band) & ~63 : 0;   // sweeps start on a 64-key tile
                const int end = std::max(m + rows, pre);
                out.push_back({base + m, rows, base + first, end - first, m - first, pre - first, band_p1});
            }
        } else {
            for (int n = 0; n < len; n += kBwdKeys) {
                const int keys = std::min(kBwdKeys, len - n);
                const int first = n < pre ? 0 : n & ~31;                          // unit slices start on 32 rows
                const int end = band >= 0 ? (int)std::min<int64_t>(len, (int64_t)n + keys + band) : len;
                out.push_back({base + n, keys, base + first, end - first, first - n, pre - n, band_p1});
            }
        }
    }
}

int check_segments(const int32_t* cu, int n_seg, int causal, int band, const int32_t* prefix) {
    if (!cu || n_seg < 0) return lv_fail(LV_EINVAL, "cu_seqlens is null or n_seg < 0");
    for (int i = 0; i < n_seg; ++i)
        if (cu[0] < 0 || cu[i + 1] < cu[i]) return lv_fail(LV_EINVAL, "cu_seqlens must start at 0 or above and not decrease (entry %d)", i);
    if (band >= 0 && (!causal || prefix)) return lv_fail(LV_EINVAL, "a band goes with the causal rule and without a prefix");
    if (prefix && !causal) return lv_fail(LV_EINVAL, "a prefix goes with the causal rule");
    for (int i = 0; prefix && i < n_seg; ++i)
        if (prefix[i] < 0) return lv_fail(LV_EINVAL, "prefix_lens[%d] = %d < 0", i, prefix[i]);
    return 0;
}

int build(const std::vector<Sweep>& base, int piece, bool backward, int32_t* desc, int max_blocks, int32_t* comb, int max_comb, int* n_comb,
          int* ws_rows) {
    struct Out { int32_t v[LV_DESC_INTS]; int64_t work; };
    const int block = backward ? kBwdKeys : kFwdRows;
    std::vector<Out> items;
    int64_t ws = 0;
    int nc = 0;
    for (const Sweep& b : base) {
        const int np = (piece > 0 && b.bn > piece) ? (b.bn + piece - 1) / piece : 1;
        if (comb) {
            if (nc >= max_comb) return lv_fail(LV_ESIZE, "room for %d combine entries", max_comb);
            const int32_t c[4] = {b.a0, b.an, (int32_t)ws, np};
            memcpy(comb + 4 * (size_t)nc, c, sizeof(c));
        }
        ++nc;
        for (int p = 0; p < np; ++p) {
            const int cut = piece > 0 ? p * piece : 0;
            const int len = piece > 0 ? std::min(piece, b.bn - cut) : b.bn;
            Out o{};
            // a forward piece starts `cut` keys later (keys counted from there), a backward piece `cut` rows later
            const int shift = backward ? b.shift + cut : b.shift - cut;
            const int prefix = backward ? b.prefix : b.prefix - cut;
            const int32_t v[LV_DESC_INTS] = {b.a0, b.an, b.b0 + cut, len, shift, piece > 0 ? (int32_t)(ws - b.a0) : 0, b.band_p1, prefix};
            memcpy(o.v, v, sizeof(v));
            o.work = (int64_t)b.an * len;
            items.push_back(o);
            ws += block;
            if (ws > 0x7fffffffLL) return lv_fail(LV_ESIZE, "too many workspace rows");
        }
    }
    if (n_comb) *n_comb = nc;
    if (ws_rows) *ws_rows = (int)ws;
    if (desc) {
        if ((int64_t)items.size() > max_blocks) return lv_fail(LV_ESIZE, "need %lld block descriptors, room for %d", (long long)items.size(), max_blocks);
        std::stable_sort(items.begin(), items.end(), [](const Out& a, const Out& b) { return a.work > b.work; });
        for (size_t i = 0; i < items.size(); ++i) memcpy(desc + i * LV_DESC_INTS, items[i].v, sizeof(items[i].v));
    }
    return (int)items.size();
}

int check_rule(int d, int hq, int hkv, float softmax_scale, float softcap, const float* slopes) {
    if (!(softcap >= 0.f) || softcap > 1e30f) return lv_fail(LV_EINVAL, "softcap %g must be a finite number above 0 (0: no cap)", (double)softcap);
    if (!(softmax_scale > -1e30f && softmax_scale < 1e30f)) return lv_fail(LV_EINVAL, "softmax_scale is not finite");
    if (slopes && hq / hkv > 64) return lv_fail(LV_EINVAL, "slopes: %d query heads per KV head (at most 64)", hq / hkv);
    return 0;
}

}  // namespace

ScoreRule lv_score_rule(float scale, float softcap, const float* slopes) {
    ScoreRule r;
    // (finite whatever the two are: a raw product of 0 stays 0)
    r.cap_in = softcap > 0.f ? (float)std::clamp(2.0 * 1.4426950408889634 * (double)scale / (double)softcap, -3e38, 3e38) : 0.f;
    r.cap_out = softcap * 1.4426950408889634f;
    r.plus0 = softcap > LV_SCORE_WIDE_CAP ? 0.f : r.cap_out;
    r.slopes = slopes;
    return r;
}
int lv_score_mod(float softcap, const float* slopes) {
    if (softcap > LV_SCORE_WIDE_CAP) return LV_SCORE_RULE | LV_SCORE_CAP | LV_SCORE_BIAS | LV_SCORE_WIDE;
    return LV_SCORE_RULE | (softcap > 0.f ? LV_SCORE_CAP : 0) | (slopes ? LV_SCORE_BIAS : 0);
}

extern "C" int lv_build_score_blocks(const int32_t* cu, int n_seg, int causal, int band, const int32_t* prefix_host, int backward, int piece,
                                     int32_t* desc, int max_blocks, int32_t* comb, int max_comb, int* n_comb, int* ws_rows) {
    try {
        if (int e = check_segments(cu, n_seg, causal, band, prefix_host)) return e;
        if (piece < 0 || piece % (backward ? 32 : 64)) return lv_fail(LV_EINVAL, "piece length %d", piece);
        std::vector<Sweep> base;
        sweeps_of(cu, n_seg, causal, band, prefix_host, backward != 0, base);
        return build(base, piece, backward != 0, desc, max_blocks, comb, max_comb, n_comb, ws_rows);
    } catch (const std::exception& e) {
        return lv_fail(LV_ESIZE, "lv_build_score_blocks: %s", e.what());
    }
}

extern "C" int lv_plan_score_split(const int32_t* cu, int n_seg, int causal, int band, const int32_t* prefix_host, int backward, int hq, int hkv,
                                   int n_cu) {
    try {
        if (int e = check_segments(cu, n_seg, causal, band, prefix_host)) return e;
        if (hq <= 0 || hkv <= 0 || hq % hkv || n_cu <= 0) return lv_fail(LV_EINVAL, "heads %d / %d, %d compute units", hq, hkv, n_cu);
        std::vector<Sweep> base;
        sweeps_of(cu, n_seg, causal, band, prefix_host, backward != 0, base);
        std::vector<int> len;
        for (const Sweep& b : base) len.push_back(b.bn);
        // fixed cost of a work item in swept elements, as for plain attention (lv_plan_fwd_split / lv_plan_bwd_split)
        const int group = hq / hkv;
        return backward ? lv_plan_sweeps(len.data(), (int)len.size(), hkv, n_cu, (128 + group - 1) / group, 256)
                        : lv_plan_sweeps(len.data(), (int)len.size(), hq, n_cu, 512, 256);
    } catch (const std::exception& e) {
        return lv_fail(LV_ESIZE, "lv_plan_score_split: %s", e.what());
    }
}

// delta = rowsum dO O with O to 16 bits of mantissa (out + its cut-off byte): dS = P (dP - delta) takes the difference of two
// numbers that a rounding of O to bf16 alone would move by more than dS's own rounding.  D / 8 threads per (row, head).
template <int D>
__global__ __launch_bounds__(256) void lv_score_delta_kernel(const __bf16* __restrict__ o, const uint8_t* __restrict__ o_lo, const __bf16* __restrict__ dout,
                                                             float* __restrict__ delta, int64_t total, int hq, int64_t o_rs, int64_t o_hs,
                                                             int64_t do_rs, int64_t do_hs, int64_t lse_stride) {
    constexpr int CPR = D / 8;
    const int64_t idx = blockIdx.x * 256ll + threadIdx.x, at = idx < total ? idx : total - 1;
    const int ch = (int)(at % CPR);
    const int64_t rh = at / CPR, row = rh / hq;
    const int head = (int)(rh % hq);
    const u32x4 a = *reinterpret_cast<const u32x4*>(o + row * o_rs + (int64_t)head * o_hs + ch * 8);
    const u32x2 lo = *reinterpret_cast<const u32x2*>(o_lo + at * 8);
    const bf16x8 b = *reinterpret_cast<const bf16x8*>(dout + row * do_rs + (int64_t)head * do_hs + ch * 8);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        s += lv_join_low((a[i >> 1] >> (16 * (i & 1))) & 0xffffu, (lo[i >> 2] >> (8 * (i & 3))) & 0xffu) * (float)b[i];
#pragma unroll
    for (int off = CPR / 2; off > 0; off >>= 1) s += __shfl_xor(s, off);
    if (ch == 0 && idx < total) delta[(int64_t)head * lse_stride + row] = s;
}

// out / lse / cut-off bytes of a row = the log-sum-exp merge of its block's pieces, first piece first, from fp32 partials
template <int D>
__global__ __launch_bounds__(256) void lv_score_combine_kernel(const float* __restrict__ ws_out, const float* __restrict__ ws_lse, __bf16* __restrict__ out,
                                                               uint8_t* __restrict__ out_lo, float* __restrict__ lse, const int32_t* __restrict__ comb,
                                                               int hq, int64_t ws_lse_stride, int64_t o_rs, int64_t o_hs, int64_t lse_stride) {
    constexpr int ROWS = 32, CPR = D / 8;
    const int e = blockIdx.x / (kFwdRows / ROWS), head = blockIdx.y;
    const int out_row0 = comb[4 * e], rows = comb[4 * e + 1], ws_row0 = comb[4 * e + 2], np = comb[4 * e + 3];
    const int r0 = blockIdx.x % (kFwdRows / ROWS) * ROWS, r1 = min(rows, r0 + ROWS);
    for (int idx = threadIdx.x; idx < (r1 - r0) * CPR; idx += 256) {
        const int row = r0 + idx / CPR, ch = idx % CPR;
        const float* lp = ws_lse + (int64_t)head * ws_lse_stride + ws_row0 + row;
        float m = -INFINITY;
        for (int p = 0; p < np; ++p) m = fmaxf(m, lp[(int64_t)p * kFwdRows]);
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, tot = 0.f;
        if (m > -INFINITY)
            for (int p = 0; p < np; ++p) {
                const float w = __expf(lp[(int64_t)p * kFwdRows] - m);
                const float* src = ws_out + ((ws_row0 + (int64_t)p * kFwdRows + row) * hq + head) * D + ch * 8;
                const f32x4 a = *reinterpret_cast<const f32x4*>(src), b = *reinterpret_cast<const f32x4*>(src + 4);
                tot += w;
#pragma unroll
                for (int i = 0; i < 4; ++i) { acc[i] += w * a[i]; acc[4 + i] += w * b[i]; }
            }
        const float inv = tot > 0.f ? 1.f / tot : 0.f;
        bf16x8 o;
        u32x2 lo = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = acc[i] * inv;
            o[i] = (__bf16)x;
            lo[i >> 2] |= lv_low_byte(x) << (8 * (i & 3));
        }
        *reinterpret_cast<bf16x8*>(out + (int64_t)(out_row0 + row) * o_rs + (int64_t)head * o_hs + ch * 8) = o;
        if (out_lo) *reinterpret_cast<u32x2*>(out_lo + ((int64_t)(out_row0 + row) * hq + head) * D + ch * 8) = lo;
        if (ch == 0) lse[(int64_t)head * lse_stride + out_row0 + row] = tot > 0.f ? m + __logf(tot) : -INFINITY;
    }
}

// dq, dk and dv = the sums of their blocks' fp32 pieces, first piece first, all three in one launch (three launches of 7 us each
// before, a twelfth of a training step of 8,192 rows at 5 / 1 heads): 32 rows of one (block, head) per workgroup, the
// workgroups of dq first
struct SumPart { const float* ws; __bf16* out; const int32_t* comb; int blk, heads; int64_t o_rs, o_hs; };
template <int D>
__global__ __launch_bounds__(256) void lv_score_combine_grads_kernel(SumPart pq, SumPart pk, SumPart pv, int n_q, int n_k) {
    constexpr int ROWS = 32, CPR = D / 8;
    int at = blockIdx.x;
    const SumPart p = at < n_q ? pq : (at < n_q + n_k ? pk : pv);
    at -= at < n_q ? 0 : (at < n_q + n_k ? n_q : n_q + n_k);
    const int chunks = p.blk / ROWS, head = at % p.heads, e = at / p.heads / chunks;
    const int out_row0 = p.comb[4 * e], rows = p.comb[4 * e + 1], ws_row0 = p.comb[4 * e + 2], np = p.comb[4 * e + 3];
    const int r0 = at / p.heads % chunks * ROWS, r1 = min(rows, r0 + ROWS);
    for (int idx = threadIdx.x; idx < (r1 - r0) * CPR; idx += 256) {
        const int row = r0 + idx / CPR, ch = idx % CPR;
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int i = 0; i < np; ++i) {
            const float* src = p.ws + ((ws_row0 + (int64_t)i * p.blk + row) * p.heads + head) * D + ch * 8;
            const f32x4 a = *reinterpret_cast<const f32x4*>(src), b = *reinterpret_cast<const f32x4*>(src + 4);
#pragma unroll
            for (int x = 0; x < 4; ++x) { acc[x] += a[x]; acc[4 + x] += b[x]; }
        }
        bf16x8 o;
#pragma unroll
        for (int x = 0; x < 8; ++x) o[x] = (__bf16)acc[x];
        *reinterpret_cast<bf16x8*>(p.out + (int64_t)(out_row0 + row) * p.o_rs + (int64_t)head * p.o_hs + ch * 8) = o;
    }
}

extern "C" int lvattn_score_combine_grads(const float* dq_ws, const float* dk_ws, const float* dv_ws, void* dq, void* dk, void* dv, const int32_t* qcomb_dev,
                                          int n_qcomb, const int32_t* kcomb_dev, int n_kcomb, int hq, int hkv, int d, int64_t dq_rs, int64_t dq_hs,
                                          int64_t dk_rs, int64_t dk_hs, int64_t dv_rs, int64_t dv_hs, void* stream) {
    if (!dq_ws || !dk_ws || !dv_ws || !dq || !dk || !dv || !qcomb_dev || !kcomb_dev) return lv_fail(LV_EINVAL, "lvattn_score_combine_grads: null pointer");
    if (n_qcomb < 0 || n_kcomb < 0 || hq <= 0 || hkv <= 0 || (d != 64 && d != 128) || ((dq_rs | dq_hs | dk_rs | dk_hs | dv_rs | dv_hs) & 7) ||
        (((uintptr_t)dq_ws | (uintptr_t)dk_ws | (uintptr_t)dv_ws | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15))
        return lv_fail(LV_EINVAL, "lvattn_score_combine_grads: sizes, strides or alignment");
    const int64_t nq = (int64_t)n_qcomb * (kFwdRows / 32) * hq, nk = (int64_t)n_kcomb * (kBwdKeys / 32) * hkv;
    if (nq + 2 * nk > 0x7fffffffLL) return lv_fail(LV_EINVAL, "grid too large");
    if (nq + nk == 0) return LV_OK;
    const SumPart q{dq_ws, (__bf16*)dq, qcomb_dev, kFwdRows, hq, dq_rs, dq_hs}, k{dk_ws, (__bf16*)dk, kcomb_dev, kBwdKeys, hkv, dk_rs, dk_hs},
        v{dv_ws, (__bf16*)dv, kcomb_dev, kBwdKeys, hkv, dv_rs, dv_hs};
    const dim3 grid((unsigned)(nq + 2 * nk));
    if (d == 128) hipLaunchKernelGGL(lv_score_combine_grads_kernel<128>, grid, dim3(256), 0, (hipStream_t)stream, q, k, v, (int)nq, (int)nk);
    else hipLaunchKernelGGL(lv_score_combine_grads_kernel<64>, grid, dim3(256), 0, (hipStream_t)stream, q, k, v, (int)nq, (int)nk);
    return hipGetLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "combine launch failed");
}

extern "C" int lvattn_score_delta(const void* out, const uint8_t* out_lo, const void* dout, float* delta, int rows, int hq, int d, int64_t o_rs, int64_t o_hs,
                                  int64_t do_rs, int64_t do_hs, int64_t lse_stride, void* stream) {
    if (!out || !out_lo || !dout || !delta) return lv_fail(LV_EINVAL, "lvattn_score_delta: null pointer");
    if (d != 64 && d != 128) return lv_fail(LV_EINVAL, "head dim %d not supported (64 or 128)", d);
    if ((((uintptr_t)out | (uintptr_t)dout) & 15) || ((uintptr_t)out_lo & 7)) return lv_fail(LV_EINVAL, "lvattn_score_delta: out / dout must be 16-byte, out_lo 8-byte aligned");
    if ((o_rs | o_hs | do_rs | do_hs) & 7) return lv_fail(LV_EINVAL, "strides must be multiples of 8 elements");
    if (rows < 0 || hq <= 0 || lse_stride < rows) return lv_fail(LV_EINVAL, "bad sizes");
    if (rows == 0) return LV_OK;
    const int64_t total = (int64_t)rows * hq * (d / 8), grid = (total + 255) / 256;
    if (grid > 0x7fffffffLL) return lv_fail(LV_EINVAL, "grid too large");
    if (d == 128) hipLaunchKernelGGL(lv_score_delta_kernel<128>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, (const __bf16*)out, out_lo, (const __bf16*)dout,
                                     delta, total, hq, o_rs, o_hs, do_rs, do_hs, lse_stride);
    else hipLaunchKernelGGL(lv_score_delta_kernel<64>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, (const __bf16*)out, out_lo, (const __bf16*)dout,
                            delta, total, hq, o_rs, o_hs, do_rs, do_hs, lse_stride);
    return hipGetLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "delta launch failed");
}

extern "C" int lvattn_score_combine(const float* ws_out, const float* ws_lse, void* out, uint8_t* out_lo, float* lse, const int32_t* comb_dev, int n_comb,
                                    int hq, int d, int64_t ws_lse_stride, int64_t o_rs, int64_t o_hs, int64_t lse_stride, void* stream) {
    if (!ws_out || !ws_lse || !out || !lse || !comb_dev) return lv_fail(LV_EINVAL, "lvattn_score_combine: null pointer");
    if (n_comb < 0 || hq <= 0 || hq > 65535 || (d != 64 && d != 128) || ((o_rs | o_hs) & 7) || (((uintptr_t)ws_out | (uintptr_t)out) & 15) || ((uintptr_t)out_lo & 7))
        return lv_fail(LV_EINVAL, "lvattn_score_combine: sizes, strides or alignment");
    if ((int64_t)n_comb * 8 > 0x7fffffffLL) return lv_fail(LV_EINVAL, "grid too large");
    if (n_comb == 0) return LV_OK;
    const dim3 grid((unsigned)(n_comb * (kFwdRows / 32)), (unsigned)hq);
    if (d == 128) hipLaunchKernelGGL(lv_score_combine_kernel<128>, grid, dim3(256), 0, (hipStream_t)stream, ws_out, ws_lse, (__bf16*)out, out_lo, lse, comb_dev, hq,
                                     ws_lse_stride, o_rs, o_hs, lse_stride);
    else hipLaunchKernelGGL(lv_score_combine_kernel<64>, grid, dim3(256), 0, (hipStream_t)stream, ws_out, ws_lse, (__bf16*)out, out_lo, lse, comb_dev, hq, ws_lse_stride,
                            o_rs, o_hs, lse_stride);
    return hipGetLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "combine launch failed");
}

extern "C" int lvattn_fwd_score(const void* q, const void* k, const void* v, void* out, uint8_t* out_lo, int out_f32, float* lse, const int32_t* desc_dev, int n_blocks,
                                int q_rows_total, int k_rows_total, int hq, int hkv, int d, int64_t q_rs, int64_t q_hs, int64_t k_rs, int64_t k_hs,
                                int64_t v_rs, int64_t v_hs, int64_t o_rs, int64_t o_hs, int64_t lse_stride, float softmax_scale, float softcap,
                                const float* slopes, void* stream) {
    if (int e = lv_check_qkv(q, k, v, hq, hkv, d, q_rs, q_hs, k_rs, k_hs, v_rs, v_hs)) return e;
    if (int e = check_rule(d, hq, hkv, softmax_scale, softcap, slopes)) return e;
    if (!out || !lse || !desc_dev) return lv_fail(LV_EINVAL, "null out/lse/desc pointer");
    if (((uintptr_t)out & (out_f32 ? 15 : 7)) || (o_rs & 3) || (o_hs & 3)) return lv_fail(LV_EINVAL, "out must be 8-byte (fp32: 16-byte) aligned with strides %% 4 == 0");
    if (out_f32 && (out_lo || o_hs != d || o_rs != (int64_t)hq * d)) return lv_fail(LV_EINVAL, "fp32 results are contiguous and have no cut-off bytes");
    if ((uintptr_t)out_lo & 15) return lv_fail(LV_EINVAL, "out_lo must be 16-byte aligned");
    if (n_blocks < 0 || q_rows_total <= 0 || k_rows_total <= 0) return lv_fail(LV_EINVAL, "bad sizes");
    if (n_blocks == 0) return LV_OK;
    if ((int64_t)n_blocks * hq > 0x7fffffffLL) return lv_fail(LV_EINVAL, "grid too large");
    FwdParams p{};
    p.q = (const __bf16*)q; p.k = (const __bf16*)k; p.v = (const __bf16*)v; p.o = (__bf16*)out; p.lse = lse;
    p.o_f32 = out_f32 ? (float*)out : nullptr; p.o_lo = out_lo;
    p.desc = (const AttnDesc*)desc_dev;
    p.n_blocks = n_blocks; p.hq = hq; p.hkv = hkv; p.group = hq / hkv;
    p.q_rows_total = q_rows_total; p.k_rows_total = k_rows_total;
    p.q_rs = q_rs; p.q_hs = q_hs; p.k_rs = k_rs; p.k_hs = k_hs; p.v_rs = v_rs; p.v_hs = v_hs;
    p.o_rs = o_rs; p.o_hs = o_hs; p.lse_stride = lse_stride;
    p.scale = softmax_scale; p.scale_log2e = softmax_scale * 1.4426950408889634f;
    if (!(fabsf(p.scale_log2e) >= 1e-20f)) p.scale_log2e = 1e-20f;   // the kernel divides slopes by it; scores this small are 0 beside them
    p.score = lv_score_rule(softmax_scale, softcap, slopes);
    if (lv_launch_fwd_pp_score(p, d, lv_score_mod(softcap, slopes), (hipStream_t)stream))
        return lv_fail(LV_ELAUNCH, "forward launch failed: %s", hipGetErrorString(hipGetLastError()));
    return LV_OK;
}

extern "C" int lvattn_bwd_score(const void* q, const void* k, const void* v, const void* dout, const float* lse, const float* delta, void* dq, void* dk,
                                void* dv, const int32_t* qdesc_dev, int n_qblocks, const int32_t* kdesc_dev, int n_kblocks, int q_rows_total,
                                int k_rows_total, int hq, int hkv, int d, int64_t q_rs, int64_t q_hs, int64_t k_rs, int64_t k_hs, int64_t v_rs,
                                int64_t v_hs, int64_t do_rs, int64_t do_hs, int64_t dq_rs, int64_t dq_hs, int64_t dk_rs, int64_t dk_hs,
                                int64_t dv_rs, int64_t dv_hs, int64_t lse_stride, float softmax_scale, float softcap, const float* slopes,
                                int accum_f32, void* stream) {
    if (int e = lv_check_qkv(q, k, v, hq, hkv, d, q_rs, q_hs, k_rs, k_hs, v_rs, v_hs)) return e;
    if (int e = check_rule(d, hq, hkv, softmax_scale, softcap, slopes)) return e;
    if (!dout || !lse || !delta || !dq || !dk || !dv) return lv_fail(LV_EINVAL, "null pointer");
    if ((n_qblocks > 0 && !qdesc_dev) || (n_kblocks > 0 && !kdesc_dev)) return lv_fail(LV_EINVAL, "null descriptor pointer");
    if (((uintptr_t)dout & 15) || ((do_rs | do_hs) & 7)) return lv_fail(LV_EINVAL, "dout must be 16-byte aligned, strides %% 8 == 0");
    if (do_rs < 0 || do_rs * 2 * 256 > 0x7fffffffLL) return lv_fail(LV_EINVAL, "dout row stride %lld elements out of range", (long long)do_rs);
    if ((((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) || ((dq_rs | dq_hs | dk_rs | dk_hs | dv_rs | dv_hs) & 3))
        return lv_fail(LV_EINVAL, "dq/dk/dv must be 16-byte aligned with strides %% 4 == 0");
    if (n_qblocks < 0 || n_kblocks < 0 || q_rows_total <= 0 || k_rows_total <= 0 || lse_stride < q_rows_total) return lv_fail(LV_EINVAL, "bad sizes");
    if (accum_f32 < 0 || accum_f32 > 2) return lv_fail(LV_EINVAL, "accum_f32 = %d (0 bf16 results, 1 fp32 added to, 2 fp32 stored)", accum_f32);
    if ((int64_t)n_qblocks * hq > 0x7fffffffLL || (int64_t)n_kblocks * hkv > 0x7fffffffLL) return lv_fail(LV_EINVAL, "grid too large");
    BwdParams p{};
    p.q = (const __bf16*)q; p.k = (const __bf16*)k; p.v = (const __bf16*)v; p.dout = (const __bf16*)dout;
    p.lse = lse; p.delta = delta; p.dq = dq; p.dk = dk; p.dv = dv;
    p.desc = (const AttnDesc*)kdesc_dev; p.qdesc = (const AttnDesc*)qdesc_dev;
    p.n_blocks = n_kblocks; p.n_qblocks = n_qblocks; p.hq = hq; p.hkv = hkv; p.group = hq / hkv;
    p.q_rows_total = q_rows_total; p.k_rows_total = k_rows_total;
    p.q_rs = q_rs; p.q_hs = q_hs; p.k_rs = k_rs; p.k_hs = k_hs; p.v_rs = v_rs; p.v_hs = v_hs;
    p.do_rs = do_rs; p.do_hs = do_hs; p.dq_rs = dq_rs; p.dq_hs = dq_hs;
    p.dk_rs = dk_rs; p.dk_hs = dk_hs; p.dv_rs = dv_rs; p.dv_hs = dv_hs;
    p.lse_stride = lse_stride; p.scale = softmax_scale; p.scale_log2e = softmax_scale * 1.4426950408889634f;
    p.f32_store = (accum_f32 == 2);
    p.score = lv_score_rule(softmax_scale, softcap, slopes);
    const int mod = lv_score_mod(softcap, slopes);
    // the two launches write different tensors and read the same ones: any order
    if (lv_launch_bwd_dkdv_rs_score(p, d, accum_f32 != 0, mod, (hipStream_t)stream) || lv_launch_bwd_dq_pp_score(p, d, accum_f32 != 0, mod, (hipStream_t)stream))
        return lv_fail(LV_ELAUNCH, "backward launch failed: %s", hipGetErrorString(hipGetLastError()));
    return LV_OK;
}
