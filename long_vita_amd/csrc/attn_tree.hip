// Attention of drafted tokens over a KV cache for gfx950: n tokens per sequence (one: an ordinary decode step), every one
// seeing the sequence's cached keys and, among the drafted keys behind them, itself and its ancestors.
//
//   keys of sequence b: cache rows [0, len_b) visible to all its tokens, row len_b + j visible to token i iff j is i or an
//   ancestor of i;  t as in attn_score.hip with token i at position len_b + depth_i;  O = softmax(t) V
//
// All query rows of one KV head -- n tokens x the group's heads -- share that head's keys, so they are the 32-wide column
// blocks of S^T = K Q^T and O^T += V^T P^T (32x32x16 MFMAs).  A workgroup is WR x WK waves: WR of them side by side over 32 WR
// query rows (32, 64 or 128), WK over the keys, 32 or 64 of every 128-key tile each.  The WR waves of a key slice share its rows of
// K and V in LDS, brought by direct global -> LDS loads into a ring of tiles that keeps 64 - 96 KB per compute unit on their
// way; a tile costs one barrier (none with WR = 1, where every wave streams for itself).  The key waves are joined once, at
// the end.  Two waves per SIMD (WR > 1) put one's exponentials beside the other's matrix products.  Few rows are bound by the
// cache's bytes, many (row blocks of 128, side by side on one XCD's L2) by the matrix and vector pipes.
//
// The keys of ALL sequences form one list of tiles, dealt evenly to G workgroups per KV head: a workgroup's share may begin
// inside one sequence and end inside another, so ragged lengths leave no compute unit waiting.  A share's result for a sequence
// goes to partial slot g + s (the pairs (g, s) along the list only ever step forward, so the sum is unique) and a second kernel
// joins a sequence's slots in order.
//
// With 128 rows per workgroup and heads of 128 the registers do not hold everything: 9 to 28 vector registers spill, outside the
// tile loop.
//
// Measured: 64 tokens over 131,000 keys, 40 / 8 heads, 225 us (763 TFLOP/s; three blocks of 128 rows for 320 rows and 10 shares each
// leave 16 of the 256 compute units without work); 8 tokens over 1,040,000 keys, 5 / 1 heads, 105 us
// (5.1 TB/s); one token over 1,048,576 keys, 40 / 8 heads, 718 us (6.0 TB/s); 25 tokens over 8 caches of 0 to 16,001 keys 63 us.
#include "cache_list.h"
#include "../../include/lvattn.h"

#include <algorithm>
#include <type_traits>

// [slots of K / V tiles][cum][lens][par][depth][anc][stat]
#define LV_TREE_LDS_FIXED (LV_TREE_MAX_BATCH * 8 + LV_TREE_MAX_TOKENS * 8 + LV_TREE_MAX_TOKENS * (LV_TREE_MAX_TOKENS / 32) * 4 + 3072)
#define LV_TREE_RING (128 * 1024)

template <int WR>
struct TreeShape {
    static constexpr int WK = WR == 4 ? 2 : 4;
    static constexpr int SUB = WR == 4 ? 2 : 1;   // 32-key slices per key wave and tile
    static constexpr int TILE = 32 * WK * SUB;    // keys per tile: 128
    static_assert(TILE == 128, "tree_plan counts tiles of 128 keys");
    static constexpr int THREADS = 64 * WR * WK;
    // tiles that taking up another sequence costs (list_scan); 0 / 3 / 5 / 8 measured: 77 / 65 / 63 / 62 us for 25 tokens of 8
    // sequences of 0 to 16K keys, 111 / 107 / 108 / 112 us for 8 tokens of 16 sequences of 40 to 30K
    static constexpr int LEAD = WR == 4 ? 5 : 3;
    template <int D> static constexpr int slot_bytes() { return TILE * 2 * D * 2; }       // a tile of K and V
    template <int D> static constexpr int slots() { return WR == 4 ? 2 : (LV_TREE_RING / slot_bytes<D>() > 4 ? 4 : LV_TREE_RING / slot_bytes<D>()); }
    template <int D> static constexpr int lds_bytes() { return slots<D>() * slot_bytes<D>() + LV_TREE_LDS_FIXED; }
};

template <int D, int WR, int MOD>
__global__ __launch_bounds__(TreeShape<WR>::THREADS, 2) void lv_tree_kernel(TreeParams p) {
    constexpr int WK = TreeShape<WR>::WK;
    constexpr int BN = TreeShape<WR>::TILE;
    constexpr int NT = TreeShape<WR>::THREADS;
    constexpr int NW = WR * WK;
    constexpr int SUB = TreeShape<WR>::SUB;
    constexpr int WN = 32;                // keys per slice
    constexpr int KS = D / 16;
    constexpr int MT = D / 32;
    constexpr int ROWB = D * 2;
    constexpr int SLICEB = WN * ROWB;     // K or V rows of one key slice
    constexpr int SLOTB = TreeShape<WR>::template slot_bytes<D>();            // a tile: [slice][K rows, V rows]
    constexpr int NS = TreeShape<WR>::template slots<D>();                    // ring slots: 2 or 4
    static_assert(SLOTB == WK * SUB * 2 * SLICEB && NS >= 2, "ring layout");
    constexpr int CPR = D / 8;
    constexpr int RPP = 64 / CPR;         // rows per 1-KiB request
    constexpr int NP = SLICEB / 1024;     // requests per K or V slice: 8 (d = 128) or 4
    constexpr int NPW = 2 * SUB * NP / WR;        // requests per wave and tile
    constexpr bool PP = WR == 4;          // ping-pong: key waves 0 and 1, the two waves of a SIMD, one phase apart
    constexpr float RESCALE_LOG2 = 8.0f;
    constexpr float OPTIMISTIC_MAX = 4096.0f;

    extern __shared__ __attribute__((aligned(16))) char smem[];
    int* const cum = reinterpret_cast<int*>(smem + NS * SLOTB);         // [LV_TREE_MAX_BATCH]
    int* const lens = cum + LV_TREE_MAX_BATCH;                          // [LV_TREE_MAX_BATCH]
    int* const par = lens + LV_TREE_MAX_BATCH;                          // [LV_TREE_MAX_TOKENS]
    int* const depth = par + LV_TREE_MAX_TOKENS;                        // [LV_TREE_MAX_TOKENS]
    uint32_t* const anc = reinterpret_cast<uint32_t*>(depth + LV_TREE_MAX_TOKENS);   // [tokens][words]: a token and its ancestors
    float* const stat = reinterpret_cast<float*>(anc + LV_TREE_MAX_TOKENS * (LV_TREE_MAX_TOKENS / 32));   // [3][8 waves][32]
    f32x4* const obuf = reinterpret_cast<f32x4*>(smem);                 // the join's buffer is the ring: [wave][MT][4][lane]
    static_assert(NS * SLOTB >= NW * MT * 4096, "the join fits the ring");

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = w % WR, wk = w / WR;
    const int r = lane & 31;
    const int h = lane >> 5;
    const int words = (p.n + 31) >> 5;

    // the row blocks of one (KV head, share) unit take consecutive slots of one XCD: they stream the same tiles
    const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
    const int rb = slot % p.n_rb;
    const int unit = (slot / p.n_rb) * 8 + xcd;
    if (unit >= p.hkv * p.shares) return;
    const int kvh = unit % p.hkv, g = unit / p.hkv;

    constexpr int LEAD = TreeShape<WR>::LEAD;
    list_scan<BN, LEAD>(p.cache_lens, p.batch, p.rows, p.n, cum, lens);
    const ListDeal deal(p.shares, __builtin_amdgcn_readfirstlane(cum[p.batch - 1]));
    if (g >= (int)deal.G) return;
    int tile = __builtin_amdgcn_readfirstlane(deal.first(g));
    const int tile_end = __builtin_amdgcn_readfirstlane(deal.first(g + 1));
    int s = 0;
    while (__builtin_amdgcn_readfirstlane(cum[s]) <= tile) ++s;

    // ---- requests: this wave's part (NPW requests, K or V rows) of its key slice, tile after tile of the sequence at hand
    int rq_s = 0, rq_t = 0, rq_t1 = 0, rq_keys = 0;      // sequence, next tile to ask for, the share's last of it, keys
    lds_char* const ring = (lds_char*)smem + wk * SUB * 2 * SLICEB;     // this wave's slices in slot 0
    const uint32_t ring_addr = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)ring);
    // one operand's rows as this wave asks for them: position -> chunk of the LDS image (the swizzle is an involution and
    // repeats every 16 rows)
    constexpr int NV = 16 / RPP;
    struct Rows { const __bf16* base; int64_t bs, rs; int voff[NV]; };
    auto rows_of = [&](const __bf16* base, int64_t bs, int64_t rs, int64_t hs) __attribute__((always_inline)) {
        Rows x{base + (int64_t)kvh * hs, bs, rs, {}};
#pragma unroll
        for (int j = 0; j < NV; ++j)
            x.voff[j] = lane / CPR * (int)(rs * 2) + list_lds_off<D>(RPP * j + lane / CPR, lane % CPR) - (RPP * j + lane / CPR) * ROWB;
        return x;
    };
    const bool v_part = WR > 1 && (wr & 1);          // WR > 1: even row waves bring K, odd ones V
    const Rows own = rows_of(v_part ? p.v : p.k, v_part ? p.v_bs : p.k_bs, v_part ? p.v_rs : p.k_rs, v_part ? p.v_hs : p.k_hs);
    const Rows own_v = WR == 1 ? rows_of(p.v, p.v_bs, p.v_rs, p.v_hs) : own;
    auto request_slice = [&](const Rows& x, uint32_t dst, int u) __attribute__((always_inline)) {
        int first = rq_t * BN + WN * (wk * SUB + u);
        // (ping-pong multiplies every slice: one behind the last key repeats it)
        if constexpr (PP) first = min(first, rq_keys - 1);
        const int valid = rq_t < rq_t1 ? min(rq_keys - first, WN) : 0;
        // nothing to bring: zero records, every lane out of range
        const uint32_t rec = valid > 0 ? (uint32_t)((valid - 1) * x.rs * 2 + ROWB) : 0u;
        const __bf16* src = x.base + (valid > 0 ? (int64_t)rq_s * x.bs + (int64_t)first * x.rs : 0);
        auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(src), 0, rec, 0x00020000);
        const int rs2 = (int)(x.rs * 2);
        if (valid <= 0 || valid >= WN) {
#pragma unroll
            for (int j = 0; j < NP; ++j) list_dma16(rsrc, x.voff[j % NV] + RPP * j * rs2, dst + j * 1024);
        } else {                                     // rows past the last key repeat it: never bytes that are no key's
            const int lr = lane / CPR;
#pragma unroll
            for (int j = 0; j < NP; ++j) list_dma16(rsrc, x.voff[j % NV] + (min(RPP * j + lr, valid - 1) - lr) * rs2, dst + j * 1024);
        }
    };
    static_assert(WR == 1 ? SUB == 1 : 2 * SUB == WR, "WR > 1: every wave brings one slice's K or V rows");
    auto request = [&](int sl) __attribute__((always_inline)) {
        const int u = wr >> 1;
        const uint32_t dst = ring_addr + sl * SLOTB + (WR == 1 ? 0 : u * 2 * SLICEB);
        request_slice(own, dst + (v_part ? SLICEB : 0), WR == 1 ? 0 : u);
        if constexpr (WR == 1) request_slice(own_v, dst + SLICEB, 0);
        ++rq_t;
    };

    int k_off[KS];     // K row read: row r, chunk 2ks + h
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k_off[ks] = list_lds_off<D>(r, 2 * ks + h);
    const int i16 = lane & 15, q4 = i16 >> 2, p4 = i16 & 3, gl = (lane >> 4) & 1;
    int v_off[MT][2];  // V transposed read
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int jh = 0; jh < 2; ++jh)
            v_off[mt][jh] = SLICEB + list_lds_off<D>(8 * jh + 4 * h + q4, 4 * mt + 2 * gl + (p4 >> 1)) + 8 * (p4 & 1);

    // this lane's query row: row -> (token, head of the group)
    const int n_rows = p.n * p.group;
    const int row = 32 * (WR * rb + wr) + r;
    const int rowc = min(row, n_rows - 1);
    const int token = rowc / p.group, head = kvh * p.group + rowc % p.group;
    float nslope2 = 0.f;
    if constexpr ((MOD & LV_SCORE_BIAS) != 0) nslope2 = lv_slope2<MOD>(p.score, head);
    const float c = MOD != 0 ? 1.f : p.scale_log2e;

    while (tile < tile_end) {
        // ---------------- one sequence of this share ----------------
        const int len = __builtin_amdgcn_readfirstlane(lens[s]), keys = len + p.n;
        const int list0 = (s ? __builtin_amdgcn_readfirstlane(cum[s - 1]) : 0) + list_lead<LEAD>(s);
        tile = max(tile, list0);
        const int t0 = tile - list0, t1 = min(tile_end, __builtin_amdgcn_readfirstlane(cum[s])) - list0;
        if (t1 <= t0) break;              // the share ends ahead of the sequence's first tile
        const bool sees_tree = t1 * BN > len;

        // WR = 1 asks for tile t + NS when its own slot is free, WR = 2 for tile t + NS - 1 behind the barrier of tile t, the
        // ping-pong for K of tile t + 2 and V of tile t + 1 in the vector phase of tile t
        rq_s = s;
        rq_t = t0;
        rq_t1 = t1;
        rq_keys = keys;
        int sl = 0;                       // slot of the tile being consumed
        if constexpr (PP) {
            static_assert(!PP || NS == 2, "two slots");
            request(0);
            if (!v_part) request(1);
        } else {
#pragma unroll
            for (int i = 0; i < (WR == 1 ? NS : NS - 1); ++i) request(i);
        }

        bf16x8 qf[KS];
        const __bf16* qptr = p.q + (int64_t)s * p.q_bs + (int64_t)token * p.q_ns + (int64_t)head * p.q_hs + 8 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(qptr + 16 * ks);

        int my_depth = token;             // without parents the tokens are a chain
        bool live = row < n_rows;
        if (p.parents) {
            list_tree(p.parents + (int64_t)s * p.parents_bs, p.n, words, sees_tree, par, depth, anc, tid, NT);
            my_depth = depth[token];
            live = live && par[token] != LV_TREE_UNUSED;
        }

        f32x16 oacc[MT];
        float m_run = -1e30f, l_run = 0.f;
        // the sum of P as it was rounded divides O, so that the rounding of a row's largest P cancels (out's error against 64 bits
        // 0.0023 -> 0.0020; not with WR = 4, whose vector phase it would lengthen by 6 %)
        constexpr bool PV_SUM = WR < 4;
        float l_pv = 0.f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 16; ++i) oacc[mt][i] = 0.f;
        // every ordinary load (and store of the sequence before) retires here: from now on the counter holds requests only
        asm volatile("" : "+v"(nslope2));
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            asm volatile("" : "+v"(qf[ks]));
            if (!live) qf[ks] = bf16x8{};      // a row that holds no token: whatever is there stays out
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

        // ---- the scores of this wave's slices of tile t (first key kb0) -> P
        f32x16 x[SUB];
        bf16x8 pf[SUB][2];     // P rounds to bf16, the matrix pipe's type; its sum is taken before the rounding
        auto weigh = [&]() __attribute__((always_inline)) {      // P against the running maximum; its row sum (this lane's half)
            const float mc = m_run * c;
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float pv = fast_exp2(__builtin_fmaf(x[u][i], c, -mc));
                    sum += pv;
                    pf[u][i >> 3][i & 7] = (__bf16)pv;
                }
            return sum;
        };
        auto softmax = [&](int kb0, bool masked) __attribute__((always_inline)) {
            if constexpr (MOD != 0) {                // t (log2 units) from the raw products
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    const int jl = kb0 + WN * u + 4 * h;
                    const float fq = (float)(len + my_depth - jl);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float dist = fq - (float)((i & 3) + 8 * (i >> 2));
                        if constexpr ((MOD & LV_SCORE_BIAS) != 0)
                            if (masked && p.parents) {       // a drafted key stands at its depth, not at its row
                                const int j = jl + (i & 3) + 8 * (i >> 2) - len;
                                if (j >= 0) dist = (float)(my_depth - depth[min(j, p.n - 1)]);
                            }
                        x[u][i] = lv_score<MOD>(x[u][i], p.scale_log2e, p.score, nslope2, dist);
                    }
                }
            }
            // Optimistic pass (see attn_fwd_pp.hip): with a finite running maximum P is formed against it without looking for
            // the tile's own; a score far above it shows as a large sum and sends the tile through the exact pass.
            bool exact = masked || __any(m_run < -1e29f);
            if (!exact) {
                const float sum = weigh();
                if (__any(!(sum <= OPTIMISTIC_MAX))) exact = true;      // (also catches inf / nan)
                else l_run += sum;
            }
            auto add_pv = [&]() __attribute__((always_inline)) {
                if constexpr (PV_SUM)
#pragma unroll
                    for (int u = 0; u < SUB; ++u) l_pv = add_bf16x8(pf[u][1], add_bf16x8(pf[u][0], l_pv));
            };
            if (!exact) { add_pv(); return; }
            if (masked) {
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    // bit e of `vis`: key kb0 + 32 u + e visible to this lane's token
                    uint32_t vis;
                    const int j0 = kb0 + WN * u - len;          // first key of the slice, counted from the first drafted one
                    if (p.parents) {
                        const uint32_t* aw = anc + token * words;
                        const int lo = j0 >> 5;        // (arithmetic shift: below 0 for a slice that starts in the cache)
                        const uint32_t a0 = lo < 0 ? 0xffffffffu : (lo < words ? aw[lo] : 0u);
                        const uint32_t a1 = lo + 1 < 0 ? 0xffffffffu : (lo + 1 < words ? aw[lo + 1] : 0u);
                        vis = (uint32_t)((((uint64_t)a1 << 32) | a0) >> (j0 & 31));
                    } else {
                        const int last = token - j0;   // keys up to the token's own
                        vis = last >= 31 ? 0xffffffffu : (last < 0 ? 0u : (2u << last) - 1u);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int e = (i & 3) + 8 * (i >> 2) + 4 * h;
                        x[u][i] = (vis >> e) & 1 ? x[u][i] : -INFINITY;
                    }
                }
            }
            float mx = x[0][0];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[u][i]);
            mx = pair32_max(mx);
            const float m_new = fmaxf(m_run, mx);
            const bool grow = (m_new - m_run) * c > RESCALE_LOG2;
            if (__any(grow)) {
                const float alpha = fast_exp2((m_run - m_new) * c);
                m_run = m_new;
                l_run *= alpha;
                l_pv *= alpha;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) oacc[mt][i] *= alpha;
            }
            l_run += weigh();
            add_pv();
        };
        // rows of unused slots hold whatever was there: zero, so that not even a NaN gets through P = 0 (every wave that shares
        // the slice writes the same zeros before it reads)
        auto blank_unused = [&](lds_char* vrows, int first) __attribute__((always_inline)) {
            const int vrow = lane >> 1;
            const int j = min(first + vrow, keys - 1) - len;
            if (j >= 0 && par[j] == LV_TREE_UNUSED)
#pragma unroll
                for (int i = 0; i < CPR / 2; ++i)
                    *(LDS_PTR(u32x4, vrows + vrow * ROWB + ((lane & 1) * (CPR / 2) + i) * 16)) = u32x4{0, 0, 0, 0};
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        };

        if constexpr (PP) {
            // Vector phase of tile t: softmax, requests.  Matrix phase: S of tile t + 1 and O^T += V_t^T P_t.  Key wave 1 runs one
            // barrier behind key wave 0, so a SIMD has one of its two waves in each phase (see attn_fwd_pp.hip).
            asm volatile("s_barrier" ::: "memory");          // (the counter is at zero: everyone's first K and V are there)
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[u][i] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const bf16x8 kf = *(LDS_PTR(bf16x8, ring + sl * SLOTB + u * 2 * SLICEB + k_off[ks]));
                    x[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ks], x[u], 0, 0, 0);
                }
            }
            // every row wave has read its K of this tile before one of them asks for the tile that replaces it
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (wk == 1) asm volatile("s_barrier" ::: "memory");
            for (int t = t0; t < t1; ++t) {
                const int kb0 = t * BN + WN * SUB * wk;
                const bool masked = kb0 + WN * SUB > len;
                softmax(kb0, masked);
                request((wr & 1) ? sl ^ 1 : sl);         // V of tile t + 1, K of tile t + 2
                __builtin_amdgcn_sched_barrier(0);
                // all but the newest requests have landed: K of tile t + 1, V of tile t
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NPW) : "memory");
                __builtin_amdgcn_sched_barrier(0);
                lds_char* const kb = ring + (sl ^ 1) * SLOTB;
                lds_char* const vb = ring + sl * SLOTB;
                if (masked && p.parents)
#pragma unroll
                    for (int u = 0; u < SUB; ++u) blank_unused(vb + u * 2 * SLICEB + SLICEB, kb0 + WN * u);
                __builtin_amdgcn_s_setprio(2);
                // groups (u, s2) of MT products with V rows 16 s2 .. of slice u and KS / 2 steps of S[u]; the fragments of a group
                // are read while the one before it runs
                bf16x8 vfr[2][MT], kfr[2][KS / 2];
                auto load_group = [&](int g, int set) __attribute__((always_inline)) {
                    const int u = g >> 1, s2 = g & 1;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, vb + v_off[mt][0] + u * 2 * SLICEB + 16 * s2 * ROWB));
                        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, vb + v_off[mt][1] + u * 2 * SLICEB + 16 * s2 * ROWB));
                        bf16x8& vf = vfr[set][mt];
                        vf[0] = lo[0]; vf[1] = lo[1]; vf[2] = lo[2]; vf[3] = lo[3];
                        vf[4] = hi[0]; vf[5] = hi[1]; vf[6] = hi[2]; vf[7] = hi[3];
                    }
#pragma unroll
                    for (int kk = 0; kk < KS / 2; ++kk) kfr[set][kk] = *(LDS_PTR(bf16x8, kb + u * 2 * SLICEB + k_off[s2 * (KS / 2) + kk]));
                };
                constexpr int RPG = 2 * MT + KS / 2, MPG = MT + KS / 2;
                static_assert(MT == KS / 2 && RPG * 2 == MPG * 3, "three reads per two products");
                load_group(0, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, RPG, 0);
#pragma unroll
                for (int g4 = 0; g4 < 2 * SUB; ++g4) {
                    const int u = g4 >> 1, s2 = g4 & 1, set = g4 & 1;
                    if (g4 + 1 < 2 * SUB) load_group(g4 + 1, set ^ 1);
                    if (s2 == 0) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[u][i] = 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {       // two accumulation targets in turn
                        oacc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vfr[set][i], pf[u][s2], oacc[i], 0, 0, 0);
                        x[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kfr[set][i], qf[s2 * (KS / 2) + i], x[u], 0, 0, 0);
                    }
                    if (g4 + 1 < 2 * SUB) {
#pragma unroll
                        for (int i = 0; i < MPG / 2; ++i) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                        }
                    } else {
                        __builtin_amdgcn_sched_group_barrier(0x008, MPG, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(0);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                sl ^= 1;
                ++tile;
            }
            if (wk == 0) asm volatile("s_barrier" ::: "memory");
        } else {
        for (int t = t0; t < t1; ++t) {
            const int kb0 = t * BN + WN * SUB * wk;
            const bool masked = kb0 + WN * SUB > len;      // drafted keys, or rows past the end, are among the wave's
            lds_char* const kb = ring + sl * SLOTB;
            if constexpr (WR == 1) {
                // K of this tile: requested before its V and the NS - 1 tiles behind it
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((2 * NS - 1) * NP) : "memory");
            } else {
                // this wave's part of the tile has landed; behind the barrier everyone's has, and everyone is done with the
                // tile before, whose slot takes the next request
                asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 2) * NPW) : "memory");
                request(sl == 0 ? NS - 1 : sl - 1);
            }
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[u][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    const bf16x8 kf = *(LDS_PTR(bf16x8, kb + u * 2 * SLICEB + k_off[ks]));
                    x[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ks], x[u], 0, 0, 0);
                }
            softmax(kb0, masked);
            if constexpr (WR == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((2 * NS - 2) * NP) : "memory");   // V of this tile
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                if (kb0 + WN * u >= keys) continue;            // (nothing was brought for a slice without keys)
                lds_char* const vb = kb + u * 2 * SLICEB;
                if (masked && p.parents) blank_unused(vb + SLICEB, kb0 + WN * u);
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, vb + v_off[mt][0] + 16 * s2 * ROWB));
                        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, vb + v_off[mt][1] + 16 * s2 * ROWB));
                        bf16x8 vf;
                        vf[0] = lo[0]; vf[1] = lo[1]; vf[2] = lo[2]; vf[3] = lo[3];
                        vf[4] = hi[0]; vf[5] = hi[1]; vf[6] = hi[2]; vf[7] = hi[3];
                        oacc[mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[u][s2], oacc[mt], 0, 0, 0);
                    }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // this wave is done with the slot
            if constexpr (WR == 1) request(sl);
            sl = sl + 1 == NS ? 0 : sl + 1;
            ++tile;
        }
        }

        // ---------------- join the key waves; this share's result for the sequence -> partial slot g + s ----------------
        // (a sequence that is the share's alone is finished here, and the second kernel passes its rows by; WR = 4 has no
        // registers left for it: a 64-token tree over 131K keys took 231 instead of 226 us)
        const bool whole = WR < 4 && p.direct && t0 == 0 && list0 + t1 == __builtin_amdgcn_readfirstlane(cum[s]);
        const int64_t part = ((int64_t)(kvh * p.n_rb + rb) * p.slots + g + s) * (32 * WR) + 32 * wr;
        int row_o = lane & 31;            // (derived anew: not kept in registers through the loop)
        asm volatile("" : "+v"(row_o));
        row_o += 32 * (WR * rb + wr);
        const int rowc_o = min(row_o, n_rows - 1), token_o = rowc_o / p.group, head_o = kvh * p.group + rowc_o % p.group;
        __bf16* const orow = p.o + (int64_t)s * p.o_bs + (int64_t)token_o * p.o_ns + (int64_t)head_o * p.o_hs;
        const float unit2 = MOD != 0 ? 0.6931471805599453f : p.scale;
        const float l_w = pair32_sum(l_run);
        if (h == 0) {
            stat[w * 32 + r] = m_run;
            stat[256 + w * 32 + r] = l_w;
        }
        if constexpr (PV_SUM) {
            const float l_x = pair32_sum(l_pv);
            if (h == 0) stat[512 + w * 32 + r] = l_x;
        }
        // (what was asked for past the share's last tile of the sequence brings nothing, but has to be over before the ring is
        // written by hand)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        float m_tot = -1e30f, l_tot = 0.f;
#pragma unroll
        for (int i = 0; i < WK; ++i) m_tot = fmaxf(m_tot, stat[(i * WR + wr) * 32 + r]);
#pragma unroll
        for (int i = 0; i < WK; ++i) l_tot += stat[256 + (i * WR + wr) * 32 + r] * fast_exp2((stat[(i * WR + wr) * 32 + r] - m_tot) * c);
        const float sc = fast_exp2((m_run - m_tot) * c);
        float l_o = l_tot;
        if constexpr (PV_SUM) {
            l_o = 0.f;
#pragma unroll
            for (int i = 0; i < WK; ++i) l_o += stat[512 + (i * WR + wr) * 32 + r] * fast_exp2((stat[(i * WR + wr) * 32 + r] - m_tot) * c);
        }
        const float inv = (l_tot > 0.f && live) ? 1.f / l_o : 0.f;
        if (wk == 0 && h == 0) {
            const float x = (l_tot > 0.f && live) ? m_tot * unit2 + __logf(l_tot) : -INFINITY;
            if (!whole) p.part_lse[part + r] = x;
            else if (p.lse && row_o < n_rows) p.lse[((int64_t)s * p.n + token_o) * p.hq + head_o] = x;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4)
                obuf[((w * MT + mt) * 4 + g4) * 64 + lane] = f32x4{oacc[mt][4 * g4] * sc, oacc[mt][4 * g4 + 1] * sc, oacc[mt][4 * g4 + 2] * sc, oacc[mt][4 * g4 + 3] * sc};
        __syncthreads();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4 / WK; ++e) {        // key wave wk finishes 16 / WK of a lane's accumulators
                const int g4 = wk * (4 / WK) + e;
                f32x4 acc = obuf[((wr * MT + mt) * 4 + g4) * 64 + lane];
#pragma unroll
                for (int i = 1; i < WK; ++i) acc += obuf[(((i * WR + wr) * MT + mt) * 4 + g4) * 64 + lane];
                acc = inv > 0.f ? acc * inv : f32x4{0.f, 0.f, 0.f, 0.f};
                const int col = 32 * mt + 8 * g4 + 4 * h;
                if (!whole) *reinterpret_cast<f32x4*>(p.part_o + (part + r) * D + col) = acc;
                else if (row_o < n_rows) *reinterpret_cast<bf16x4*>(orow + col) = bf16x4{(__bf16)acc[0], (__bf16)acc[1], (__bf16)acc[2], (__bf16)acc[3]};
            }
        __syncthreads();                  // the next sequence's requests go where obuf is
        ++s;
    }
}

// out / lse of a row = the log-sum-exp merge of its sequence's slots; every sum has a fixed order.  D / 4 threads take a slot's
// columns; the 1024 / D groups of them share one row's slots (ONE_ROW: few rows) or take a row each (many).
template <int D, int WR, bool ONE_ROW>
__global__ __launch_bounds__(256) void lv_tree_join_kernel(TreeParams p) {
    constexpr int rows_pb = 32 * WR;
    constexpr int TPR = D / 4;                // threads per slot row
    constexpr int GR = 256 / TPR;             // groups
    __shared__ int cum[LV_TREE_MAX_BATCH];
    __shared__ float wgt[ONE_ROW ? LV_TREE_MAX_SHARES : 1];
    __shared__ float red[8];
    __shared__ f32x4 osum[GR][TPR];
    const int tid = threadIdx.x, gr = tid / TPR, col = tid % TPR * 4;
    list_scan<TreeShape<WR>::TILE, TreeShape<WR>::LEAD>(p.cache_lens, p.batch, p.rows, p.n, cum, nullptr);
    const ListDeal deal(p.shares, cum[p.batch - 1]);
    const int n_rows = p.n * p.group;
    const int64_t total = (int64_t)p.batch * p.hkv * n_rows;
    for (int64_t idx = ONE_ROW ? blockIdx.x : (int64_t)blockIdx.x * GR + gr; idx < total; idx += ONE_ROW ? total : (int64_t)gridDim.x * GR) {   // (sequence, KV head, row)
    const int row = (int)((uint32_t)idx % n_rows), unit = (int)((uint32_t)idx / n_rows), kvh = unit % p.hkv, s = unit / p.hkv;
    const int g0 = deal.share_of(s ? cum[s - 1] + list_lead<TreeShape<WR>::LEAD>(s) : 0), g1 = deal.share_of(cum[s] - 1);
    const int rb = row / rows_pb;
    const int64_t part = ((int64_t)(kvh * p.n_rb + rb) * p.slots + g0 + s) * rows_pb + row % rows_pb;
    const int np = g1 - g0 + 1;               // at most shares
    if (np == 1 && p.direct) continue;        // the share that had the sequence to itself wrote the result (uniform where barriers follow)
    const float* lp = p.part_lse + part;
    const float* po = p.part_o + part * D + col;
    float m = -INFINITY, tot = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if constexpr (ONE_ROW) {
        for (int i = tid; i < np; i += 256) {
            const float x = lp[(int64_t)i * rows_pb];
            wgt[i] = x;
            m = fmaxf(m, x);
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
        if ((tid & 63) == 0) red[tid >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        for (int i = tid; i < np; i += 256) {
            const float x = m > -INFINITY ? __expf(wgt[i] - m) : 0.f;
            wgt[i] = x;
            tot += x;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) tot += __shfl_xor(tot, off);
        if ((tid & 63) == 0) red[4 + (tid >> 6)] = tot;
        __syncthreads();
        tot = red[4] + red[5] + red[6] + red[7];
#pragma unroll 4
        for (int i = gr; i < np; i += GR) acc += wgt[i] * *reinterpret_cast<const f32x4*>(po + (int64_t)i * rows_pb * D);
        osum[gr][tid % TPR] = acc;
        __syncthreads();
        if (gr > 0) return;
#pragma unroll
        for (int i = 1; i < GR; ++i) acc += osum[i][tid];
    } else {
        for (int i = 0; i < np; ++i) m = fmaxf(m, lp[(int64_t)i * rows_pb]);
        if (m > -INFINITY) {
#pragma unroll 4
            for (int i = 0; i < np; ++i) {
                const float x = __expf(lp[(int64_t)i * rows_pb] - m);
                tot += x;
                acc += x * *reinterpret_cast<const f32x4*>(po + (int64_t)i * rows_pb * D);
            }
        }
    }
    const float inv = tot > 0.f ? 1.f / tot : 0.f;
    const int token = row / p.group, head = kvh * p.group + row % p.group;
    __bf16* op = p.o + (int64_t)s * p.o_bs + (int64_t)token * p.o_ns + (int64_t)head * p.o_hs + col;
#pragma unroll
    for (int e = 0; e < 4; ++e) op[e] = (__bf16)(acc[e] * inv);
    if (p.lse && col == 0) p.lse[((int64_t)s * p.n + token) * p.hq + head] = tot > 0.f ? m + __logf(tot) : -INFINITY;
    }
}

struct TreePlan { int wr, n_rb, shares, slots; int64_t part_rows; };
// Rows per workgroup: 32, 64 or 128.  Shares per KV head: a workgroup's ring fills a compute unit's LDS, so 256 workgroups fill
// the chip, and one more would wait for a second round; never more shares than tiles.
static TreePlan tree_plan(int batch, int n, int rows, int hq, int hkv) {
    TreePlan t;
    const int n_rows = n * (hq / hkv);
    t.wr = n_rows <= 32 ? 1 : (n_rows <= 64 ? 2 : 4);
    t.n_rb = (n_rows + 32 * t.wr - 1) / (32 * t.wr);
    const int64_t tiles = (int64_t)batch * ((rows + 127) / 128);
    int64_t g = 256 / ((int64_t)hkv * t.n_rb);
    if (g > tiles) g = tiles;
    if (g < 1) g = 1;
    t.shares = (int)g;                                  // <= 256 = LV_TREE_MAX_SHARES
    t.slots = (int)g + batch - 1;
    t.part_rows = (int64_t)hkv * t.n_rb * t.slots * 32 * t.wr;
    return t;
}

template <int D, int WR>
static void launch_tree(const TreeParams& p, int mod, unsigned blocks, int64_t out_rows, hipStream_t stream) {
    const dim3 grid(blocks), block(TreeShape<WR>::THREADS);
    constexpr size_t lds = TreeShape<WR>::template lds_bytes<D>();
    static_assert(lds <= 160 * 1024, "one workgroup per compute unit");
    switch (mod) {
        case 0: hipLaunchKernelGGL((lv_tree_kernel<D, WR, 0>), grid, block, lds, stream, p); break;
        case LV_SCORE_CAP: hipLaunchKernelGGL((lv_tree_kernel<D, WR, LV_SCORE_CAP>), grid, block, lds, stream, p); break;
        case LV_SCORE_BIAS: hipLaunchKernelGGL((lv_tree_kernel<D, WR, LV_SCORE_BIAS>), grid, block, lds, stream, p); break;
        case LV_SCORE_CAP | LV_SCORE_BIAS: hipLaunchKernelGGL((lv_tree_kernel<D, WR, LV_SCORE_CAP | LV_SCORE_BIAS>), grid, block, lds, stream, p); break;
        default: hipLaunchKernelGGL((lv_tree_kernel<D, WR, LV_SCORE_CAP | LV_SCORE_BIAS | LV_SCORE_WIDE>), grid, block, lds, stream, p);
    }
    if (hipPeekAtLastError() != hipSuccess) return;   // (reported by the caller)
    // a workgroup per row takes the slots side by side; with more rows than the chip holds at once (eight workgroups to a compute
    // unit) a group of threads walks its row's slots instead, eight or sixteen rows to a workgroup at a time, and the workgroups
    // that the chip holds go round the rows (122,880 rows of 256 sequences: the list's lengths are summed 2048 times, not 15,360)
    if (out_rows <= 2048) hipLaunchKernelGGL((lv_tree_join_kernel<D, WR, true>), dim3((unsigned)out_rows), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((lv_tree_join_kernel<D, WR, false>), dim3((unsigned)std::min<int64_t>((out_rows * (D / 4) + 255) / 256, 2048)), dim3(256), 0, stream, p);
}

extern "C" int64_t lvattn_tree_workspace_bytes(int batch, int n, int rows, int hq, int hkv, int d) {
    if (batch <= 0 || n <= 0 || rows < n || hq <= 0 || hkv <= 0 || hq % hkv || (d != 64 && d != 128)) return 0;
    return tree_plan(batch, n, rows, hq, hkv).part_rows * (d + 1) * (int64_t)sizeof(float);
}

extern "C" int lvattn_tree(const void* q, const void* k, const void* v, void* out, float* lse, const int32_t* cache_lens, const int32_t* parents,
                           int64_t parents_batch_stride, void* workspace, int64_t workspace_bytes, int batch, int n, int rows, int hq, int hkv,
                           int d, int64_t q_bs, int64_t q_ns, int64_t q_hs, int64_t k_bs, int64_t k_rs, int64_t k_hs, int64_t v_bs, int64_t v_rs,
                           int64_t v_hs, int64_t o_bs, int64_t o_ns, int64_t o_hs, float softmax_scale, float softcap, const float* slopes,
                           void* stream) {
    if (q_bs < 0 || q_ns < 0 || ((q_bs | q_ns) & 7)) return lv_fail(LV_EINVAL, "lvattn_tree: q batch / token strides must be non-negative multiples of 8 elements");
    if (int e = lv_check_qkv(q, k, v, hq, hkv, d, 0, q_hs, k_rs, k_hs, v_rs, v_hs)) return e;
    if (!out || !cache_lens || !workspace) return lv_fail(LV_EINVAL, "lvattn_tree: null out / cache_lens / workspace pointer");
    if (batch <= 0 || batch > LV_TREE_MAX_BATCH) return lv_fail(LV_EINVAL, "lvattn_tree: batch %d (1 to %d)", batch, LV_TREE_MAX_BATCH);
    if (n <= 0 || n > LV_TREE_MAX_TOKENS) return lv_fail(LV_EINVAL, "lvattn_tree: %d tokens per sequence (1 to %d)", n, LV_TREE_MAX_TOKENS);
    if (rows < n) return lv_fail(LV_EINVAL, "lvattn_tree: a cache of %d rows cannot hold %d drafted tokens", rows, n);
    if (((k_bs | v_bs) & 7) || k_bs < 0 || v_bs < 0) return lv_fail(LV_EINVAL, "lvattn_tree: K / V batch strides must be non-negative multiples of 8 elements");
    if (((uintptr_t)workspace & 15) || parents_batch_stride < 0) return lv_fail(LV_EINVAL, "lvattn_tree: workspace must be 16-byte aligned, the parents' stride not negative");
    if (!(softcap >= 0.f) || softcap > 1e30f) return lv_fail(LV_EINVAL, "lvattn_tree: softcap %g must be a finite number above 0 (0: no cap)", (double)softcap);
    if (!(softmax_scale > 0.f && softmax_scale < 1e30f)) return lv_fail(LV_EINVAL, "lvattn_tree: softmax_scale %g must be a finite number above 0", (double)softmax_scale);
    const TreePlan t = tree_plan(batch, n, rows, hq, hkv);
    const int64_t need = t.part_rows * (d + 1) * (int64_t)sizeof(float);
    if (workspace_bytes < need) return lv_fail(LV_ESIZE, "lvattn_tree: %lld bytes of workspace needed, room for %lld", (long long)need, (long long)workspace_bytes);
    const int64_t units = (int64_t)hkv * t.shares, blocks = (units + 7) / 8 * 8 * t.n_rb;
    const int64_t join = (int64_t)batch * hkv * n * (hq / hkv);
    if (blocks > 0x7fffffffLL || join > 0x7fffffffLL || (int64_t)batch * (rows / 128 + 16) > 0x7fffffffLL)
        return lv_fail(LV_EINVAL, "lvattn_tree: grid too large");
    TreeParams p{};
    p.q = (const __bf16*)q; p.k = (const __bf16*)k; p.v = (const __bf16*)v; p.o = (__bf16*)out; p.lse = lse;
    p.cache_lens = cache_lens; p.parents = parents; p.parents_bs = parents_batch_stride;
    p.part_o = (float*)workspace; p.part_lse = p.part_o + t.part_rows * d;
    p.batch = batch; p.n = n; p.rows = rows; p.hq = hq; p.hkv = hkv; p.group = hq / hkv;
    p.n_rb = t.n_rb; p.shares = t.shares; p.slots = t.slots;
    p.direct = t.wr < 4 && !(((uintptr_t)out & 7) || ((o_bs | o_ns | o_hs) & 3));       // results can be stored four columns at a time
    p.q_bs = q_bs; p.q_ns = q_ns; p.q_hs = q_hs; p.k_bs = k_bs; p.k_rs = k_rs; p.k_hs = k_hs; p.v_bs = v_bs; p.v_rs = v_rs; p.v_hs = v_hs;
    p.o_bs = o_bs; p.o_ns = o_ns; p.o_hs = o_hs;
    p.scale = softmax_scale; p.scale_log2e = softmax_scale * 1.4426950408889634f;
    p.score = lv_score_rule(softmax_scale, softcap, slopes);
    const int mod = LV_SCORE_BITS(lv_score_mod(softcap, slopes));
    hipStream_t st = (hipStream_t)stream;
    if (d == 128) {
        if (t.wr == 1) launch_tree<128, 1>(p, mod, (unsigned)blocks, join, st);
        else if (t.wr == 2) launch_tree<128, 2>(p, mod, (unsigned)blocks, join, st);
        else launch_tree<128, 4>(p, mod, (unsigned)blocks, join, st);
    } else {
        if (t.wr == 1) launch_tree<64, 1>(p, mod, (unsigned)blocks, join, st);
        else if (t.wr == 2) launch_tree<64, 2>(p, mod, (unsigned)blocks, join, st);
        else launch_tree<64, 4>(p, mod, (unsigned)blocks, join, st);
    }
    return hipPeekAtLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "lvattn_tree: launch failed: %s", hipGetErrorString(hipGetLastError()));
}

// ---------------------------------------------------------------------------
// The accepted path of a tree becomes the cache's new rows: row len + path[i] -> row len + i, in place, K, V and (optional)
// the accumulated weights.  path is ascending (a parent stands before its child), so i <= path[i]; one workgroup per
// (sequence, KV head) reads every row it moves before it writes any, 16 bytes per thread and step of 32 rows: the rows of a
// step lie at or above the destinations of the steps before it, never below, so later steps read what was there.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(512) void lv_tree_accept_kernel(AcceptParams p) {
    const int s = blockIdx.x / p.hkv, kvh = blockIdx.x % p.hkv;
    const int len = min(max(p.cache_lens[s], 0), p.rows - p.n);
    const int m = min(max(p.n_accept[s], 0), p.n);
    if (p.new_lens && kvh == 0 && threadIdx.x == 0) p.new_lens[s] = len + m;
    const int cpr = p.d / 8;
    const int* path = p.path + (int64_t)s * p.n;
    const int step = blockDim.x / cpr;
    __bf16* kb = p.k + (int64_t)s * p.k_bs + (int64_t)kvh * p.k_hs;
    __bf16* vb = p.v + (int64_t)s * p.v_bs + (int64_t)kvh * p.v_hs;
    for (int i0 = 0; i0 < m; i0 += step) {
        const int i = i0 + threadIdx.x / cpr, ch = threadIdx.x % cpr;
        const bool on = i < m;
        int src = 0;
        u32x4 kx{}, vx{};
        float wx = 0.f;
        if (on) {
            src = min(max(path[i], i), p.n - 1);      // an index that is out of order moves nothing below its own row
            kx = *reinterpret_cast<const u32x4*>(kb + (int64_t)(len + src) * p.k_rs + ch * 8);
            vx = *reinterpret_cast<const u32x4*>(vb + (int64_t)(len + src) * p.v_rs + ch * 8);
            if (p.weight && ch == 0) wx = p.weight[(int64_t)s * p.w_bs + (int64_t)kvh * p.w_hs + len + src];
        }
        asm volatile("" : "+v"(kx), "+v"(vx), "+v"(wx));   // the loads have returned before this thread reaches the barrier
        __syncthreads();
        if (on) {
            *reinterpret_cast<u32x4*>(kb + (int64_t)(len + i) * p.k_rs + ch * 8) = kx;
            *reinterpret_cast<u32x4*>(vb + (int64_t)(len + i) * p.v_rs + ch * 8) = vx;
            if (p.weight && ch == 0) p.weight[(int64_t)s * p.w_bs + (int64_t)kvh * p.w_hs + len + i] = wx;
        }
        __syncthreads();
    }
}

extern "C" int lv_tree_accept_lens(void* k, void* v, float* weight, const int32_t* cache_lens, const int32_t* path, const int32_t* n_accept,
                                   int32_t* new_lens, int batch, int n, int rows, int hkv, int d, int64_t k_bs, int64_t k_rs, int64_t k_hs,
                                   int64_t v_bs, int64_t v_rs, int64_t v_hs, int64_t w_bs, int64_t w_hs, void* stream) {
    if (!k || !v || !cache_lens || !path || !n_accept) return lv_fail(LV_EINVAL, "lv_tree_accept: null pointer");
    if (d != 64 && d != 128) return lv_fail(LV_EINVAL, "lv_tree_accept: head dim %d (64 or 128)", d);
    if (batch <= 0 || hkv <= 0 || n <= 0 || rows < n) return lv_fail(LV_EINVAL, "lv_tree_accept: bad sizes");
    if ((((uintptr_t)k | (uintptr_t)v) & 15) || ((k_bs | k_rs | k_hs | v_bs | v_rs | v_hs) & 7))
        return lv_fail(LV_EINVAL, "lv_tree_accept: k / v must be 16-byte aligned with strides %% 8 == 0");
    if ((int64_t)batch * hkv > 0x7fffffffLL) return lv_fail(LV_EINVAL, "lv_tree_accept: grid too large");
    AcceptParams p{};
    p.k = (__bf16*)k; p.v = (__bf16*)v; p.weight = weight; p.cache_lens = cache_lens; p.path = path; p.n_accept = n_accept; p.new_lens = new_lens;
    p.n = n; p.rows = rows; p.hkv = hkv; p.d = d;
    p.k_bs = k_bs; p.k_rs = k_rs; p.k_hs = k_hs; p.v_bs = v_bs; p.v_rs = v_rs; p.v_hs = v_hs; p.w_bs = w_bs; p.w_hs = w_hs;
    hipLaunchKernelGGL(lv_tree_accept_kernel, dim3((unsigned)(batch * hkv)), dim3(512), 0, (hipStream_t)stream, p);
    return hipGetLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "lv_tree_accept: launch failed");
}

extern "C" int lv_tree_accept(void* k, void* v, float* weight, const int32_t* cache_lens, const int32_t* path, const int32_t* n_accept, int batch,
                              int n, int rows, int hkv, int d, int64_t k_bs, int64_t k_rs, int64_t k_hs, int64_t v_bs, int64_t v_rs, int64_t v_hs,
                              int64_t w_bs, int64_t w_hs, void* stream) {
    return lv_tree_accept_lens(k, v, weight, cache_lens, path, n_accept, nullptr, batch, n, rows, hkv, d, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs, w_bs, w_hs, stream);
}
