// Attention weight received by every cached key, for gfx950: what cache eviction goes by.
//
//   w_out[kvh, j] = w_in[kvh, j] + sum over tokens i and query heads h of kvh's group of rho_i exp(t_ij - lse_ih)
//
// t and the visible keys are those of attn_tree.hip, lse comes from the attention itself, rho is an optional weight per token
// (0 for drafted tokens that were not accepted); it enters as log2(rho) beside lse, so it costs nothing per score.  One product,
// S = Q K^T, with the KEY on the lane (32x32x16 MFMA, A = query rows, B = keys): a key's sum over 32 query rows is a sum over
// its lane's 16 accumulators.  Nothing is ever summed by atomics.  Two kernels:
//
// - up to 128 query rows per KV head (a decode step, a tree), twice that in two passes: bound by K's bytes.  The query fragments and, with up to 64 rows,
//   the rows' constants stay in registers, eight waves per workgroup stream K, each its own 32-key slices through its own LDS slots by
//   direct global -> LDS loads, without a barrier; tiles of all sequences are dealt evenly (cache_list.h).  The old weight of a
//   key travels with its slice, so w_out is written on the spot.
// - more rows (a large tree, a prompt): a workgroup holds the fragments of 128 keys in registers and the query rows stream
//   through an LDS ring of 64-row tiles shared by its four waves, two on each half of the keys, on alternate 32 rows.  A
//   first small kernel prepares the rows' constants.  When there are fewer key blocks than the chip has room for, the rows
//   are cut into pieces whose sums are added in order by a last kernel.  8 MFMAs (256 cycles) stand against 16 exponentials,
//   multiply-adds and adds per 32 x 32 scores, so the vector work bounds it; few rows pay for every 128 keys' loads (125 rows
//   of the 16 ragged caches below: 192 us, streamed 68 us).
//
// Registers: the streaming kernel with four row tiles of 128 spills 16 to 57 vector registers (97 with a wide cap); with a cap and
// slopes some are reloaded inside the tile loop, and such a wait is also one for the requests on their way.  The other kernel's spills
// (5 to 7, heads of 128 without slopes) lie outside its loop.
//
// Measured, 40 / 8 heads of 128: one token over 4 caches of 7,777 to 65,536 keys 65 us (48 us streaming, 5.7 TB/s; 5 us copying
// the unused rows); a prompt of 8,191 tokens 398 us (864 TFLOP/s); trees of 25 / 32 / 51 / 64 / 128 tokens over 16 ragged caches of
// 107K keys, in place, 67 / 126 / 135 / 207 / 338 us.
#include "cache_list.h"
#include "../../include/lvattn.h"

// Direct global -> LDS load of one float per lane: lane i -> LDS byte lds_dst + 4 i
__device__ __forceinline__ void weight_dma4(const float* g, uint32_t lds_dst) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(g), "s"(lds_dst) : "memory");
}

// log2(rho) - lse log2(e) of a row, plus what lv_score_plus wants on top: what its scores' exponents start from; -inf for a row that counts for nothing
__device__ __forceinline__ float row_constant(const WeightParams& p, int s, int token, int head) {
    const float rho = p.row_weight ? p.row_weight[(int64_t)s * p.n + token] : 1.f;
    const float l = p.lse[((int64_t)s * p.n + token) * p.hq + head];
    if (!(rho > 0.f) || !(l > -INFINITY)) return -INFINITY;
    return (p.row_weight ? __builtin_amdgcn_logf(rho) : 0.f) + (p.score.plus0 - l * 1.4426950408889634f);
}

// rows that hold no key keep their weights (launched when w_out is not w_in); 1024 rows of one (sequence, KV head) per workgroup,
// four per thread, all loads on their way at once (129K rows of 8 heads: 10.2 us with sixteen per thread in 4096-row workgroups, 6.1 us so)
#define LV_WEIGHT_COPY 1024
__global__ __launch_bounds__(256) void lv_weight_copy_kernel(WeightParams p) {
    const int bh = blockIdx.y, s = bh / p.hkv, kvh = bh % p.hkv;
    const int keys = list_len(p.cache_lens, s, p.rows, p.n) + p.n;
    const int j0 = blockIdx.x * LV_WEIGHT_COPY + threadIdx.x;
    const float* src = p.w_in + (int64_t)s * p.wi_bs + (int64_t)kvh * p.wi_hs;
    float* dst = p.w_out + (int64_t)s * p.wo_bs + (int64_t)kvh * p.wo_hs;
    float x[LV_WEIGHT_COPY / 256];
#pragma unroll
    for (int i = 0; i < LV_WEIGHT_COPY / 256; ++i)
        if (j0 + 256 * i >= keys && j0 + 256 * i < p.rows) x[i] = src[j0 + 256 * i];
#pragma unroll
    for (int i = 0; i < LV_WEIGHT_COPY / 256; ++i)
        if (j0 + 256 * i >= keys && j0 + 256 * i < p.rows) dst[j0 + 256 * i] = x[i];
}

// ---------------------------------------------------------------------------
// up to 32 RT query rows
// ---------------------------------------------------------------------------
#define LV_WEIGHT_TILE 256                    // keys per tile: 32 for each of eight waves
#define LV_WEIGHT_STREAM_ROWS 128             // query rows of a pass over the keys
// Two passes at most, then the other kernel (160 / 255 rows, two passes against it: 152 / 168 against 267 / 310 us for 16 ragged caches
// of 107K keys, whose longest sets its grid, 133 / 141 against 164 / 196 us for one of 131K, 143 / 151 against 112 / 138 us for 64
// short ones; with three passes it is 210 against 209 us for the long one).
#define LV_WEIGHT_PASSES 2
template <int D> constexpr int weight_slots() { return D == 128 ? 2 : 4; }
template <int D> constexpr int weight_slot_bytes() { return 32 * D * 2 + 256; }        // a slice of K, the 32 old weights
template <int D> constexpr int weight_lds_bytes() {
    return 8 * weight_slots<D>() * weight_slot_bytes<D>() + LV_TREE_MAX_BATCH * 8 + LV_TREE_MAX_TOKENS * 8 + LV_TREE_MAX_TOKENS * (LV_TREE_MAX_TOKENS / 32) * 4 + 4 * LV_WEIGHT_STREAM_ROWS * 4;
}

template <int D, int RT, int MOD>
__global__ __launch_bounds__(512, 2) void lv_weight_stream_kernel(WeightParams p) {
    constexpr int KS = D / 16;
    constexpr int ROWB = D * 2;
    constexpr int CPR = D / 8;
    constexpr int RPP = 64 / CPR;             // rows per 1-KiB request
    constexpr int NP = 32 * ROWB / 1024;      // K requests per slice: 8 (d = 128) or 4
    constexpr int NV = 16 / RPP;
    constexpr int NS = weight_slots<D>();
    constexpr int SLOTB = weight_slot_bytes<D>();
    constexpr int BN = LV_WEIGHT_TILE;
    constexpr int LEAD = 3;       // (0 / 3 / 8: 48 / 44.5 / 45.5 us for 8 tokens of 16 sequences of 40 to 30K keys)

    extern __shared__ __attribute__((aligned(16))) char smem[];
    int* const cum = reinterpret_cast<int*>(smem + 8 * NS * SLOTB);     // [LV_TREE_MAX_BATCH]
    int* const lens = cum + LV_TREE_MAX_BATCH;
    int* const par = lens + LV_TREE_MAX_BATCH;                          // [LV_TREE_MAX_TOKENS]
    int* const depth = par + LV_TREE_MAX_TOKENS;
    uint32_t* const anc = reinterpret_cast<uint32_t*>(depth + LV_TREE_MAX_TOKENS);
    float* const rc = reinterpret_cast<float*>(anc + LV_TREE_MAX_TOKENS * (LV_TREE_MAX_TOKENS / 32));   // [3][SR]: constant, position, slope
    constexpr int SR = LV_WEIGHT_STREAM_ROWS;
    int* const rtok = reinterpret_cast<int*>(rc + 3 * SR);              // [SR]: token of a row

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int words = (p.n + 31) >> 5;
    const int n_rows = p.n * p.group;

    const int kvh = blockIdx.x % p.hkv, g = blockIdx.x / p.hkv;

    list_scan<BN, LEAD>(p.cache_lens, p.batch, p.rows, p.n, cum, lens);
    const ListDeal deal(p.shares, __builtin_amdgcn_readfirstlane(cum[p.batch - 1]));
    if (g >= (int)deal.G) return;
    int tile = __builtin_amdgcn_readfirstlane(deal.first(g));
    const int tile_end = __builtin_amdgcn_readfirstlane(deal.first(g + 1));
    int s = 0;
    while (__builtin_amdgcn_readfirstlane(cum[s]) <= tile) ++s;

    lds_char* const my = (lds_char*)smem + w * NS * SLOTB;
    const uint32_t my_addr = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)my);
    int voff[NV];      // this lane's part of a request: the LDS image is swizzled inside a row, which goes on the source address
#pragma unroll
    for (int j = 0; j < NV; ++j)
        voff[j] = lane / CPR * (int)(p.k_rs * 2) + list_lds_off<D>(RPP * j + lane / CPR, lane % CPR) - (RPP * j + lane / CPR) * ROWB;
    int k_off[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k_off[ks] = list_lds_off<D>(r, 2 * ks + h);

    while (tile < tile_end) {
        const int len = __builtin_amdgcn_readfirstlane(lens[s]), keys = len + p.n;
        const int list0 = (s ? __builtin_amdgcn_readfirstlane(cum[s - 1]) : 0) + list_lead<LEAD>(s);
        tile = max(tile, list0);
        const int t0 = tile - list0, t1 = min(tile_end, __builtin_amdgcn_readfirstlane(cum[s])) - list0;
        if (t1 <= t0) break;                  // the share ends ahead of the sequence's first tile
        const __bf16* const k0 = p.k + (int64_t)s * p.k_bs + (int64_t)kvh * p.k_hs;
        const float* const w0 = p.w_in + (int64_t)s * p.wi_bs + (int64_t)kvh * p.wi_hs;
        float* const wo0 = p.w_out + (int64_t)s * p.wo_bs + (int64_t)kvh * p.wo_hs;

        // a slice of K and its old weights; rows past the last key repeat it, slices past the share bring nothing of K
        auto request = [&](int t, int sl) __attribute__((always_inline)) {
            const int first = t * BN + 32 * w;
            const int valid = t < t1 ? min(keys - first, 32) : 0;
            const uint32_t rec = valid > 0 ? (uint32_t)((valid - 1) * p.k_rs * 2 + ROWB) : 0u;
            auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(k0 + (valid > 0 ? (int64_t)first * p.k_rs : 0)), 0, rec, 0x00020000);
            const int rs2 = (int)(p.k_rs * 2), lr = lane / CPR;
            const uint32_t dst = my_addr + sl * SLOTB;
            if (valid <= 0 || valid >= 32) {
#pragma unroll
                for (int j = 0; j < NP; ++j) list_dma16(rsrc, voff[j % NV] + RPP * j * rs2, dst + j * 1024);
            } else {
#pragma unroll
                for (int j = 0; j < NP; ++j) list_dma16(rsrc, voff[j % NV] + (min(RPP * j + lr, valid - 1) - lr) * rs2, dst + j * 1024);
            }
            weight_dma4(w0 + min(first + r, keys - 1), dst + 32 * ROWB);       // (always inside: keys >= 1)
        };
#pragma unroll
        for (int i = 0; i < NS; ++i) request(t0 + i, i);

        const bool sees_tree = t1 * BN > len;
        if (p.parents) list_tree(p.parents + (int64_t)s * p.parents_bs, p.n, words, sees_tree, par, depth, anc, tid, 512);

        // query fragments (lane r: row 32 b + r), and the rows' constants in LDS
        __syncthreads();                  // the previous sequence's constants are no longer read
        if (tid < SR) {
            const int tc = min(p.row0 + tid, n_rows - 1), token = tc / p.group, head = kvh * p.group + tc % p.group;
            rc[tid] = (p.row0 + tid < n_rows && !(p.parents && par[token] == LV_TREE_UNUSED)) ? row_constant(p, s, token, head) : -INFINITY;
            if constexpr ((MOD & LV_SCORE_BIAS) != 0) {
                rc[SR + tid] = (float)(p.parents ? depth[token] : token);
                rc[2 * SR + tid] = lv_slope2<MOD>(p.score, head);
            }
            rtok[tid] = token;
        }
        bf16x8 qf[RT][KS];
#pragma unroll
        for (int b = 0; b < RT; ++b) {
            const int row = p.row0 + 32 * b + r, rowc = min(row, n_rows - 1), token = rowc / p.group;
            const __bf16* qp = p.q + (int64_t)s * p.q_bs + (int64_t)token * p.q_ns + (int64_t)(kvh * p.group + rowc % p.group) * p.q_hs + 8 * h;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qf[b][ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
        }
        // every ordinary load and store retires here: from now on the counter holds requests and the loop's stores
#pragma unroll
        for (int b = 0; b < RT; ++b)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[b][ks]));
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int b = 0; b < RT; ++b)                // a row that counts for nothing may hold anything
            if (!(rc[32 * b + r] > -INFINITY))
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) qf[b][ks] = bf16x8{};

        int sl = 0;
        for (int t = t0; t < t1; ++t) {
            const int kb0 = t * BN + 32 * w, key = kb0 + r;
            lds_char* const kb = my + sl * SLOTB;
            // this slice has landed when no more than the slices behind it are on their way (the loop's stores, in between, only
            // make the wait a little longer than it has to be)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * (NP + 1)) : "memory");
            if (kb0 < keys) {
                // two row tiles' products side by side; four row tiles, whose fragments fill the registers, go one after the other and
                // read the slice four times
                constexpr int XT = RT <= 2 ? RT : 1;
                f32x16 x[XT];
                auto products = [&](int b0) __attribute__((always_inline)) {
#pragma unroll
                    for (int b = 0; b < XT; ++b)
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[b][i] = 0.f;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        const bf16x8 kf = *(LDS_PTR(bf16x8, kb + k_off[ks]));
#pragma unroll
                        for (int b = 0; b < XT; ++b) x[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf[b0 + b][ks], kf, x[b], 0, 0, 0);
                    }
                };
                products(0);
                const float old = *(LDS_PTR(float, kb + 32 * ROWB + 4 * r));
                const bool masked = kb0 + 32 > len;
                const int jt = key - len;
                // positions count from the sequence's length: exact where it matters, also in caches of more than 2^24 keys
                float kpos = (float)jt;
                if constexpr ((MOD & LV_SCORE_BIAS) != 0)
                    if (p.parents && jt >= 0 && jt < p.n) kpos = (float)depth[jt];
                float sum = 0.f;
                int row_of = 4 * h;       // (with four row tiles the constants are read from LDS every time: the registers are full)
                if constexpr (RT > 2) asm volatile("" : "+v"(row_of));
#pragma unroll
                for (int b = 0; b < RT; ++b) {
                    if (XT == 1 && b > 0) {
                        __builtin_amdgcn_sched_barrier(0);
                        products(b);
                    }
                    const f32x16& xb = x[XT == 1 ? 0 : b];
                    float pv[16];
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4) {
                        const int ar = 32 * b + 8 * q4 + row_of;     // rows of accumulators 4 q4 .. + 3
                        const f32x4 cc = *reinterpret_cast<const f32x4*>(rc + ar);
                        f32x4 pos = {}, slope = {};
                        if constexpr ((MOD & LV_SCORE_BIAS) != 0) {
                            pos = *reinterpret_cast<const f32x4*>(rc + SR + ar);
                            slope = *reinterpret_cast<const f32x4*>(rc + 2 * SR + ar);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int i = 4 * q4 + e;
                            float t2;
                            if constexpr (MOD != 0) t2 = lv_score_plus<MOD>(xb[i], p.scale_log2e, p.score, slope[e], pos[e] - kpos, cc[e]);
                            else t2 = __builtin_fmaf(xb[i], p.scale_log2e, cc[e]);
                            pv[i] = fast_exp2(t2);
                        }
                    }
                    if (masked) {
                        // a chain: row R (token R / group) sees drafted key jt from row jt * group on; a tree's keys are looked up
                        const int first_row = key >= keys ? 0x7fffffff : max(jt, 0) * p.group;
                        const bool look = p.parents && key < keys && jt >= 0;
                        int row_m = 4 * h;
                        asm volatile("" : "+v"(row_m));          // (the rows' tokens are looked up here, not kept)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int ar = 32 * b + (i & 3) + 8 * (i >> 2) + row_m;
                            bool vis = p.row0 + ar >= first_row;
                            if (look) vis = (anc[rtok[ar] * words + (jt >> 5)] >> (jt & 31)) & 1;
                            pv[i] = vis ? pv[i] : 0.f;
                            asm volatile("" : "+v"(pv[i]));      // keeps this a branch
                        }
                    }
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
                        for (int i = 0; i < o; ++i) pv[i] += pv[i + o];
                    sum += pv[0];
                }
                sum = pair32_sum(sum);
                if (h == 0 && key < keys) wo0[key] = old + sum;
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // this wave is done with the slot
            request(t + NS, sl);
            sl = sl + 1 == NS ? 0 : sl + 1;
            ++tile;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");            // (what was asked for past the end is over before the slots are filled anew)
        ++s;
    }
}

// ---------------------------------------------------------------------------
// more rows
// ---------------------------------------------------------------------------
#define LV_WEIGHT_KEYS 128                    // keys per workgroup
#define LV_WEIGHT_ROWS 64                     // query rows per step

// constants of the rows of (sequence, KV head): [3][rows padded to 64] = exponent offset, position behind the cache, -log2(e) slope; and, per 256
// rows, whether one of them counts for nothing
__global__ __launch_bounds__(256) void lv_weight_rows_kernel(WeightParams p) {
    __shared__ int par[LV_TREE_MAX_TOKENS], depth[LV_TREE_MAX_TOKENS];
    const int bh = blockIdx.y, s = bh / p.hkv, kvh = bh % p.hkv;
    if (p.parents) list_tree(p.parents + (int64_t)s * p.parents_bs, p.n, 0, false, par, depth, nullptr, threadIdx.x, 256);
    const int row = blockIdx.x * 256 + threadIdx.x;
    float cst = -INFINITY, pos = 0.f, slope = 0.f;
    if (row < p.n * p.group) {
        const int token = row / p.group, head = kvh * p.group + row % p.group;
        if (!(p.parents && par[token] == LV_TREE_UNUSED)) cst = row_constant(p, s, token, head);
        pos = (float)(p.parents ? depth[token] : token);
        if (p.score.slopes) slope = -1.4426950408889634f * p.score.slopes[head];
    }
    const int dead = __syncthreads_or(row < p.n * p.group && !(cst > -INFINITY));
    if (threadIdx.x == 0) p.dead[(int64_t)bh * gridDim.x + blockIdx.x] = dead ? 1u : 0u;
    if (row >= p.rows_pad) return;
    float* out = p.row_const + (int64_t)bh * 3 * p.rows_pad + row;
    out[0] = cst;
    out[p.rows_pad] = pos;
    out[2 * (int64_t)p.rows_pad] = slope;
}

// three workgroups fit a compute unit (without a tree; with one, or with the positions and slopes of a bias in registers, two)
// GUARD: rows that count for nothing (unused slots, a weight of 0, an lse of -inf) may hold anything, NaN included, so their terms are
// guarded.  Where only an lse can make such a row (no parents, no row weights), the plain kernel leaves the pieces that have any
// to a guarded launch behind it (p.rest), whose other workgroups end at once.  A prompt of 8,191 tokens, 40 / 8 heads: 392 us
// without any such care, 395 so, 411 with a test for such rows inside the loop, 450 with every term guarded.
template <int D, int MOD, bool GUARD>
__global__ __launch_bounds__(256, (MOD & LV_SCORE_BIAS) || GUARD ? 2 : 3) void lv_weight_block_kernel(WeightParams p) {
    constexpr int KS = D / 16;
    constexpr int CPR = D / 8;
    constexpr int ROWB = D * 2;
    constexpr int TR = LV_WEIGHT_ROWS;
    constexpr int RPP = 64 / CPR;
    constexpr int NP = TR * ROWB / 1024 / 4;  // Q requests per wave and step: 4 or 2
    constexpr int QB = TR * ROWB;
    constexpr int SLOTB = QB + 3 * TR * 4;    // Q rows, three constants per row
    constexpr int NS = 3;

    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* const red = reinterpret_cast<float*>(smem + NS * SLOTB);                 // [LV_WEIGHT_KEYS]
    int* const par = reinterpret_cast<int*>(red + LV_WEIGHT_KEYS);                  // [LV_TREE_MAX_TOKENS]
    int* const depth = par + LV_TREE_MAX_TOKENS;
    uint32_t* const anc = reinterpret_cast<uint32_t*>(depth + LV_TREE_MAX_TOKENS);

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kw = w & 1, rw = w >> 1;
    const int r = lane & 31, h = lane >> 5;

    // heads and sequences fastest, then row pieces, then key blocks from the first (under a causal rule the heaviest) on
    const int bh = blockIdx.x % (p.batch * p.hkv);
    const int rest = blockIdx.x / (p.batch * p.hkv);
    const int piece = rest % p.pieces, kb = rest / p.pieces;
    const int s = bh / p.hkv, kvh = bh % p.hkv;
    const int len = list_len(p.cache_lens, s, p.rows, p.n), keys = len + p.n;
    const int k0 = kb * LV_WEIGHT_KEYS;
    const float* const wi = p.w_in + (int64_t)s * p.wi_bs + (int64_t)kvh * p.wi_hs;
    float* const wo = p.w_out + (int64_t)s * p.wo_bs + (int64_t)kvh * p.wo_hs;
    if (k0 >= keys) {                     // behind the last key: the weights stay as they are
        if (piece == 0 && p.w_in != p.w_out && !p.rest)
            for (int j = k0 + tid; j < min(k0 + LV_WEIGHT_KEYS, p.rows); j += 256) wo[j] = wi[j];
        return;
    }
    const int n_rows = p.n * p.group;
    const int words = (p.n + 31) >> 5;

    // the rows that see any key of the block, this piece's share of them
    int row_lo = 0;
    if (!p.parents && k0 > len) row_lo = (k0 - len) * p.group / TR * TR;     // a chain: drafted key j is seen from token j on
    const int steps = (n_rows - row_lo + TR - 1) / TR;
    const int st0 = (int)((int64_t)steps * piece / p.pieces), st1 = (int)((int64_t)steps * (piece + 1) / p.pieces);
    if (!GUARD || p.rest) {               // (rows past the last repeat it, in its own step)
        const uint32_t* flag = p.dead + (int64_t)bh * ((p.rows_pad + 255) >> 8);
        uint32_t any = 0;
        for (int i = ((row_lo + st0 * TR) >> 8) + lane; i <= (min(row_lo + st1 * TR, n_rows) - 1) >> 8; i += 64) any |= flag[i];
        if (__any(st0 < st1 && any != 0) != GUARD) return;        // (the same in all four waves)
    }
    if (p.parents && k0 + LV_WEIGHT_KEYS > len) list_tree(p.parents + (int64_t)s * p.parents_bs, p.n, words, true, par, depth, anc, tid, 256);

    // ---- this wave's keys: two groups of 32, fragments for the whole kernel
    bf16x8 kf[2][KS];
    int key[2];
    float kpos[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int base = k0 + 64 * kw + 32 * g;
        key[g] = base + r;
        const int valid = min(max(keys - base, 0), 32);      // rows past the last key read as zero and count for nothing
        auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(p.k + (int64_t)s * p.k_bs + (int64_t)kvh * p.k_hs + (valid ? (int64_t)base * p.k_rs : 0)), 0,
                                                    valid ? (uint32_t)((valid - 1) * p.k_rs * 2 + ROWB) : 0u, 0x00020000);
        const int off = (int)(r * p.k_rs * 2) + 16 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kf[g][ks] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, off + 32 * ks, 0, 0));
        kpos[g] = (float)(key[g] - len);
        if constexpr ((MOD & LV_SCORE_BIAS) != 0)
            if (p.parents && key[g] >= len && key[g] < keys) kpos[g] = (float)depth[key[g] - len];
    }
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(kf[g][ks]));


    // ---- requests: wave w brings rows 16 w .. 16 w + 15 of a step and one of the constants' arrays.  A lane's rows move on by TR
    // per step, so their offsets from the step's first token are carried along instead of divided and multiplied for.
    const int ns2 = (int)(p.q_ns * 2), hs2 = (int)(p.q_hs * 2);
    const int step_tok = TR / p.group, step_head = TR % p.group;
    const int wrap = ns2 - p.group * hs2;                      // (a head number past the group: the next token's)
    int rq_row = row_lo + st0 * TR;                            // first row of the next step
    int tok0 = __builtin_amdgcn_readfirstlane(rq_row / p.group), g0 = __builtin_amdgcn_readfirstlane(rq_row % p.group);
    int rq_g[NP], rq_off[NP], rq_ch[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int tr = RPP * (NP * w + j) + lane / CPR;       // row of the tile
        rq_ch[j] = list_lds_off<D>(tr, lane % CPR) - tr * ROWB;
        rq_g[j] = (g0 + tr) % p.group;
        rq_off[j] = (g0 + tr) / p.group * ns2 + rq_g[j] * hs2 + rq_ch[j];
    }
    const __bf16* const q0 = p.q + (int64_t)s * p.q_bs + (int64_t)kvh * p.group * p.q_hs;
    const int which = ((MOD & LV_SCORE_BIAS) != 0 && w < 3) ? w : 0;
    const float* const c0 = p.row_const + ((int64_t)bh * 3 + which) * p.rows_pad + lane;
    const uint32_t lds_base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_char*)smem);
    auto request = [&](int sl) __attribute__((always_inline)) {
        const uint32_t dst = lds_base + sl * SLOTB;
        if (rq_row + TR <= n_rows) {
            auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(q0 + (int64_t)tok0 * p.q_ns), 0, 0x7fffffff, 0x00020000);
#pragma unroll
            for (int j = 0; j < NP; ++j) list_dma16(rs, rq_off[j], dst + (NP * w + j) * 1024);
        } else {                                               // rows past the last one repeat it (their constant is -inf)
            const int tb = min(tok0, p.n - 1);
            auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(q0 + (int64_t)tb * p.q_ns), 0, 0x7fffffff, 0x00020000);
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const int row = min(rq_row + RPP * (NP * w + j) + lane / CPR, n_rows - 1);
                list_dma16(rs, (row / p.group - tb) * ns2 + row % p.group * hs2 + rq_ch[j], dst + (NP * w + j) * 1024);
            }
        }
        weight_dma4(c0 + min(rq_row, p.rows_pad - TR), dst + QB + which * TR * 4);     // (steps past the last are never used)
        rq_row += TR;
        tok0 += step_tok;
        g0 += step_head;
        const bool over = g0 >= p.group;                       // the step's own first token moves on by one more: so do the offsets' zero
        if (over) { g0 -= p.group; ++tok0; }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            rq_g[j] += step_head;
            const bool next = rq_g[j] >= p.group;
            rq_g[j] -= next ? p.group : 0;
            rq_off[j] += step_head * hs2 + (next ? wrap : 0) - (over ? ns2 : 0);
        }
    };
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (st0 < st1) {
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) request(i);
    }

    // Who sees which key.  A chain: row R (token R / group) sees drafted key jt from row jt * group on; so a lane's key has a first
    // row, and a group of keys a row from which on every row sees all of it.  A tree's keys are looked up.
    int first_row[2], full_row[2];
    bool tree_group[2];
    uint32_t seen = 0;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int kl = k0 + 64 * kw + 32 * g + 31;            // last key of the group
        tree_group[g] = p.parents && kl >= len;
        full_row[g] = tree_group[g] || kl >= keys ? 0x7fffffff : max(kl - len, 0) * p.group;
        first_row[g] = key[g] >= keys ? 0x7fffffff : max(key[g] - len, 0) * p.group;
    }

    float sum[2] = {0.f, 0.f}, lost[2] = {0.f, 0.f};     // a key may collect tens of thousands of terms: compensated sums
    int sl = 0;
    for (int st = st0; st < st1; ++st) {
        // this wave's part of the step has landed; behind the barrier everyone's has, and everyone is done with the step before,
        // whose slot takes the next request
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 2) * (NP + 1)) : "memory");
        request(sl == 0 ? NS - 1 : sl - 1);
        lds_char* const qb = (lds_char*)smem + sl * SLOTB;
        const int row0 = row_lo + st * TR + 32 * rw;      // first row of this wave's tile
        if (row0 < n_rows) {
            f32x4 cv[4], pv4[4], sv4[4];
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                lds_char* const cp = qb + QB + (32 * rw + 8 * q4 + 4 * h) * 4;
                cv[q4] = *(LDS_PTR(f32x4, cp));
                if constexpr ((MOD & LV_SCORE_BIAS) != 0) {
                    pv4[q4] = *(LDS_PTR(f32x4, cp + TR * 4));
                    sv4[q4] = *(LDS_PTR(f32x4, cp + 2 * TR * 4));
                }
            }
            f32x16 x[2];
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[g][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const bf16x8 qf = *(LDS_PTR(bf16x8, qb + list_lds_off<D>(32 * rw + r, 2 * ks + h)));
                x[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf, kf[0][ks], x[0], 0, 0, 0);
                x[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf, kf[1][ks], x[1], 0, 0, 0);
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float pv[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float cc = cv[i >> 2][i & 3];
                    float e;
                    if constexpr (MOD != 0) {
                        float dist = 0.f, sl2 = 0.f;
                        if constexpr ((MOD & LV_SCORE_BIAS) != 0) { dist = pv4[i >> 2][i & 3] - kpos[g]; sl2 = sv4[i >> 2][i & 3]; }
                        e = lv_score_plus<MOD>(x[g][i], p.scale_log2e, p.score, sl2, dist, cc);
                    } else {
                        e = __builtin_fmaf(x[g][i], p.scale_log2e, cc);
                    }
                    pv[i] = fast_exp2(e);
                    // GUARD: rows that count for nothing may hold anything, NaN included: min(NaN, 0) = 0
                    if constexpr (GUARD) pv[i] = fminf(pv[i], cc > -INFINITY ? INFINITY : 0.f);
                }
                if (row0 < full_row[g]) {          // some row of the tile misses some key of the group
                    const int base = row0 + 4 * h;
                    if (tree_group[g]) {
                        const int jt = key[g] - len;
#pragma unroll 1
                        for (int i = 0; i < 16; ++i) {
                            const int token = min((base + (i & 3) + 8 * (i >> 2)) / p.group, p.n - 1);
                            bool vis = key[g] < keys;
                            if (vis && jt >= 0) vis = (anc[token * words + (jt >> 5)] >> (jt & 31)) & 1;
                            seen = (seen & ~(1u << i)) | ((uint32_t)vis << i);
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            pv[i] = (seen >> i) & 1 ? pv[i] : 0.f;
                            asm volatile("" : "+v"(pv[i]));      // keeps this a branch
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            pv[i] = base + (i & 3) + 8 * (i >> 2) >= first_row[g] ? pv[i] : 0.f;
                            asm volatile("" : "+v"(pv[i]));
                        }
                    }
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1)
#pragma unroll
                    for (int i = 0; i < o; ++i) pv[i] += pv[i + o];
                const float y = pv[0] - lost[g], z = sum[g] + y;
                lost[g] = (z - sum[g]) - y;
                sum[g] = z;
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        sl = sl + 1 == NS ? 0 : sl + 1;
    }
    // no request may outlive the workgroup: its LDS could already belong to another one
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    float tot[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) tot[g] = pair32_sum(sum[g] - lost[g]);
    if (rw == 1 && h == 0)
#pragma unroll
        for (int g = 0; g < 2; ++g) red[64 * kw + 32 * g + r] = tot[g];
    __syncthreads();
    if (rw == 0 && h == 0) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if (key[g] >= p.rows) continue;
            tot[g] += red[64 * kw + 32 * g + r];
            if (p.pieces > 1) {
                if (key[g] < keys) p.part[((int64_t)piece * p.batch * p.hkv + bh) * p.rows + key[g]] = tot[g];
            } else {
                wo[key[g]] = wi[key[g]] + (key[g] < keys ? tot[g] : 0.f);
            }
        }
    }
}

// w_out = w_in + the pieces' sums, first piece first
__global__ __launch_bounds__(256) void lv_weight_join_kernel(WeightParams p) {
    const int bh = blockIdx.y;
    const int s = bh / p.hkv, kvh = bh % p.hkv;
    const int j = blockIdx.x * 256 + threadIdx.x;
    const int keys = list_len(p.cache_lens, s, p.rows, p.n) + p.n;
    // blocks that begin behind the last key were copied by the kernel before
    if (j >= p.rows || j / LV_WEIGHT_KEYS * LV_WEIGHT_KEYS >= keys) return;
    float x = p.w_in[(int64_t)s * p.wi_bs + (int64_t)kvh * p.wi_hs + j];
    if (j < keys) {
        float add = 0.f;
        for (int i = 0; i < p.pieces; ++i) add += p.part[((int64_t)i * p.batch * p.hkv + bh) * p.rows + j];
        x += add;
    }
    p.w_out[(int64_t)s * p.wo_bs + (int64_t)kvh * p.wo_hs + j] = x;
}

// ---------------------------------------------------------------------------
struct WeightPlan { bool stream; int shares, pieces, key_blocks, rows_pad; int64_t part_floats, const_floats, flags; int64_t bytes() const { return 4 * (part_floats + const_floats + flags); } };
static WeightPlan weight_plan(int batch, int n, int rows, int hq, int hkv) {
    WeightPlan t{};
    const int n_rows = n * (hq / hkv);
    t.stream = n_rows <= LV_WEIGHT_PASSES * LV_WEIGHT_STREAM_ROWS && n <= LV_TREE_MAX_TOKENS && batch <= LV_TREE_MAX_BATCH;
    if (t.stream) {
        const int64_t tiles = (int64_t)batch * ((rows + LV_WEIGHT_TILE - 1) / LV_WEIGHT_TILE);
        int64_t g = 256 / hkv;                // a workgroup's slots fill a compute unit's LDS
        if (g > tiles) g = tiles;
        t.shares = (int)(g < 1 ? 1 : g);
        return t;
    }
    t.rows_pad = (n_rows + LV_WEIGHT_ROWS - 1) / LV_WEIGHT_ROWS * LV_WEIGHT_ROWS;
    t.key_blocks = (rows + LV_WEIGHT_KEYS - 1) / LV_WEIGHT_KEYS;
    // three workgroups fit a compute unit: at least twice that many, so that the heavy ones start first and the light ones fill
    // in; a piece keeps at least 8 steps so that its keys' fragments are worth fetching
    const int64_t units = (int64_t)batch * hkv * t.key_blocks;
    const int steps = t.rows_pad / LV_WEIGHT_ROWS;
    int64_t g = units >= 1536 ? 1 : (1536 + units - 1) / units;
    if (g > (steps + 7) / 8) g = (steps + 7) / 8;
    t.pieces = (int)(g < 1 ? 1 : g);
    t.part_floats = t.pieces > 1 ? (int64_t)t.pieces * batch * hkv * rows : 0;
    t.const_floats = (int64_t)batch * hkv * 3 * t.rows_pad;
    t.flags = (int64_t)batch * hkv * ((t.rows_pad + 255) / 256);
    return t;
}

template <int D>
static void launch_stream(const WeightParams& p, int mod, int rt, unsigned blocks, hipStream_t stream) {
#define LV_W(M) do { \
        if (rt == 1) hipLaunchKernelGGL((lv_weight_stream_kernel<D, 1, M>), dim3(blocks), dim3(512), weight_lds_bytes<D>(), stream, p); \
        else if (rt == 2) hipLaunchKernelGGL((lv_weight_stream_kernel<D, 2, M>), dim3(blocks), dim3(512), weight_lds_bytes<D>(), stream, p); \
        else hipLaunchKernelGGL((lv_weight_stream_kernel<D, 4, M>), dim3(blocks), dim3(512), weight_lds_bytes<D>(), stream, p); } while (0)
    static_assert(weight_lds_bytes<D>() <= 160 * 1024, "one workgroup per compute unit");
    switch (mod) {
        case 0: LV_W(0); break;
        case LV_SCORE_CAP: LV_W(LV_SCORE_CAP); break;
        case LV_SCORE_BIAS: LV_W(LV_SCORE_BIAS); break;
        case LV_SCORE_CAP | LV_SCORE_BIAS: LV_W((LV_SCORE_CAP | LV_SCORE_BIAS)); break;
        default: LV_W((LV_SCORE_CAP | LV_SCORE_BIAS | LV_SCORE_WIDE));
    }
#undef LV_W
}

template <int D>
static void launch_block(const WeightParams& p, int mod, bool guard, unsigned blocks, hipStream_t stream) {
    constexpr size_t base = (size_t)3 * (LV_WEIGHT_ROWS * D * 2 + 3 * LV_WEIGHT_ROWS * 4) + LV_WEIGHT_KEYS * 4;
    constexpr size_t tree = LV_TREE_MAX_TOKENS * 8 + LV_TREE_MAX_TOKENS * (LV_TREE_MAX_TOKENS / 32) * 4;
    static_assert(3 * base <= 160 * 1024 && 2 * (base + tree) <= 160 * 1024, "workgroups per compute unit");
    const size_t lds = base + (p.parents ? tree : 0);
#define LV_W(M) do { \
        if (guard) hipLaunchKernelGGL((lv_weight_block_kernel<D, M, true>), dim3(blocks), dim3(256), lds, stream, p); \
        else hipLaunchKernelGGL((lv_weight_block_kernel<D, M, false>), dim3(blocks), dim3(256), lds, stream, p); } while (0)
    switch (mod) {
        case 0: LV_W(0); break;
        case LV_SCORE_CAP: LV_W(LV_SCORE_CAP); break;
        case LV_SCORE_BIAS: LV_W(LV_SCORE_BIAS); break;
        case LV_SCORE_CAP | LV_SCORE_BIAS: LV_W((LV_SCORE_CAP | LV_SCORE_BIAS)); break;
        default: LV_W((LV_SCORE_CAP | LV_SCORE_BIAS | LV_SCORE_WIDE));
    }
#undef LV_W
}

extern "C" int64_t lv_key_weights_workspace_bytes(int batch, int n, int rows, int hq, int hkv) {
    if (batch <= 0 || n <= 0 || rows < n || hq <= 0 || hkv <= 0 || hq % hkv || (int64_t)n * (hq / hkv) > 0x7ffff000LL) return 0;
    return weight_plan(batch, n, rows, hq, hkv).bytes();
}

extern "C" int lv_key_weights(const void* q, const void* k, const float* lse, const float* row_weight, const float* w_in, float* w_out,
                              const int32_t* cache_lens, const int32_t* parents, int64_t parents_bs, void* workspace, int64_t workspace_bytes,
                              int batch, int n, int rows, int hq, int hkv, int d, int64_t q_bs, int64_t q_ns, int64_t q_hs, int64_t k_bs, int64_t k_rs,
                              int64_t k_hs, int64_t wi_bs, int64_t wi_hs, int64_t wo_bs, int64_t wo_hs, float softmax_scale, float softcap,
                              const float* slopes, void* stream) {
    if (q_bs < 0 || q_ns < 0 || ((q_bs | q_ns) & 7)) return lv_fail(LV_EINVAL, "lv_key_weights: q batch / token strides must be non-negative multiples of 8 elements");
    if (int e = lv_check_qkv(q, k, k, hq, hkv, d, 0, q_hs, k_rs, k_hs, k_rs, k_hs)) return e;
    if (!lse || !w_in || !w_out || !cache_lens) return lv_fail(LV_EINVAL, "lv_key_weights: null lse / weight / cache_lens pointer");
    if (batch <= 0 || n <= 0 || rows < n) return lv_fail(LV_EINVAL, "lv_key_weights: batch %d, %d tokens, %d cache rows", batch, n, rows);
    if (parents && n > LV_TREE_MAX_TOKENS) return lv_fail(LV_EINVAL, "lv_key_weights: a tree of %d tokens (at most %d)", n, LV_TREE_MAX_TOKENS);
    if ((int64_t)n * (hq / hkv) > 0x7ffff000LL) return lv_fail(LV_EINVAL, "lv_key_weights: too many query rows");
    // a step of 64 query rows is addressed with 32-bit byte offsets from its first token
    if (q_hs < 0 || (66 * q_ns + (hq / hkv) * q_hs) * 2 > 0x7fffffffLL || q_ns > 0x3fffffffLL || q_hs > 0x3fffffffLL)
        return lv_fail(LV_EINVAL, "lv_key_weights: q token / head strides %lld / %lld out of range", (long long)q_ns, (long long)q_hs);
    if (k_bs < 0 || (k_bs & 7) || parents_bs < 0) return lv_fail(LV_EINVAL, "lv_key_weights: batch strides must not be negative, K's a multiple of 8 elements");
    if (!(softcap >= 0.f) || softcap > 1e30f) return lv_fail(LV_EINVAL, "lv_key_weights: softcap %g must be a finite number above 0 (0: no cap)", (double)softcap);
    if (!(softmax_scale > -1e30f && softmax_scale < 1e30f)) return lv_fail(LV_EINVAL, "lv_key_weights: softmax_scale is not finite");
    const WeightPlan t = weight_plan(batch, n, rows, hq, hkv);
    const int64_t need = t.bytes();
    if (need && (!workspace || ((uintptr_t)workspace & 15))) return lv_fail(LV_EINVAL, "lv_key_weights: workspace must be there and 16-byte aligned");
    if (workspace_bytes < need) return lv_fail(LV_ESIZE, "lv_key_weights: %lld bytes of workspace needed, room for %lld", (long long)need, (long long)workspace_bytes);
    if ((int64_t)batch * hkv > 65535 || (int64_t)batch * (rows / LV_WEIGHT_TILE + 16) > 0x7fffffffLL) return lv_fail(LV_EINVAL, "lv_key_weights: grid too large");
    WeightParams p{};
    p.q = (const __bf16*)q; p.k = (const __bf16*)k; p.lse = lse; p.row_weight = row_weight; p.w_in = w_in; p.w_out = w_out;
    p.cache_lens = cache_lens; p.parents = parents; p.parents_bs = parents_bs;
    p.row_const = (float*)workspace; p.part = p.row_const + t.const_floats; p.dead = (uint32_t*)(p.part + t.part_floats);
    p.batch = batch; p.n = n; p.rows = rows; p.hq = hq; p.hkv = hkv; p.group = hq / hkv; p.pieces = t.pieces; p.shares = t.shares; p.rows_pad = t.rows_pad;
    p.q_bs = q_bs; p.q_ns = q_ns; p.q_hs = q_hs; p.k_bs = k_bs; p.k_rs = k_rs; p.k_hs = k_hs;
    p.wi_bs = wi_bs; p.wi_hs = wi_hs; p.wo_bs = wo_bs; p.wo_hs = wo_hs;
    p.scale_log2e = softmax_scale * 1.4426950408889634f;
    p.score = lv_score_rule(softmax_scale, softcap, slopes);
    const int mod = LV_SCORE_BITS(lv_score_mod(softcap, slopes));
    hipStream_t st = (hipStream_t)stream;
    if (t.stream) {
        const int n_rows = n * p.group, rt = n_rows <= 32 ? 1 : (n_rows <= 64 ? 2 : 4);
        if (w_in != w_out)
            hipLaunchKernelGGL(lv_weight_copy_kernel, dim3((unsigned)((rows + LV_WEIGHT_COPY - 1) / LV_WEIGHT_COPY), (unsigned)(batch * hkv)), dim3(256), 0, st, p);
        const unsigned blocks = (unsigned)(hkv * t.shares);
        for (p.row0 = 0; p.row0 < n_rows; p.row0 += LV_WEIGHT_STREAM_ROWS) {
            if (d == 128) launch_stream<128>(p, mod, rt, blocks, st);
            else launch_stream<64>(p, mod, rt, blocks, st);
            p.w_in = w_out; p.wi_bs = wo_bs; p.wi_hs = wo_hs;      // the next pass adds to what this one left
        }
    } else {
        const int64_t blocks = (int64_t)batch * hkv * t.key_blocks * t.pieces;
        if (blocks > 0x7fffffffLL) return lv_fail(LV_EINVAL, "lv_key_weights: grid too large");
        hipLaunchKernelGGL(lv_weight_rows_kernel, dim3((unsigned)((t.rows_pad + 255) / 256), (unsigned)(batch * hkv)), dim3(256), 0, st, p);
        const bool guard = parents || row_weight;
        for (p.rest = 0; p.rest < (guard ? 1 : 2); ++p.rest) {
            if (d == 128) launch_block<128>(p, mod, guard || p.rest, (unsigned)blocks, st);
            else launch_block<64>(p, mod, guard || p.rest, (unsigned)blocks, st);
        }
        if (t.pieces > 1)
            hipLaunchKernelGGL(lv_weight_join_kernel, dim3((unsigned)((rows + 255) / 256), (unsigned)(batch * hkv)), dim3(256), 0, st, p);
    }
    return hipGetLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "lv_key_weights: launch failed");
}
