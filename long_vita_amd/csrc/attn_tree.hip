// Attention of drafted tokens over a KV cache for gfx950: n tokens per sequence (one: an ordinary decode step), every one
// seeing the sequence's cached keys and, among the drafted keys behind them, itself and its ancestors.
//
//   keys of sequence b: cache rows [0, len_b) visible to all its tokens, row len_b + j visible to token i iff j is i or an
//   ancestor of i;  t as in attn_score.hip with token i at position len_b + depth_i;  O = softmax(t) V
//
// All query rows of one KV head -- n tokens x the group's heads -- share that head's keys, so they are the 32-wide column
// blocks of S^T = K Q^T and O^T += V^T P^T (32x32x16 MFMAs) and each K / V byte is read once for all of them.  A workgroup is
// 4 waves on a tile of 128 keys: WR of them side by side over up to 32 WR query rows, 4 / WR over the tile's keys (few rows:
// the waves split the keys and are joined through LDS at the end; many rows: every wave sweeps the whole tile).
//
// Few rows are bound by the cache's bytes, many by the matrix products.  The keys of ALL sequences form one list of tiles,
// dealt evenly to G workgroups per KV head: a workgroup's share may begin inside one sequence and end inside another, so
// ragged lengths leave no compute unit waiting.  Its result for a sequence goes to partial slot g + s (the pairs (g, s) along
// the list only ever step forward, so the sum is unique) and a second kernel joins a sequence's slots in order.
#include "internal.h"
#include "../../include/lvattn.h"

typedef __attribute__((address_space(3))) char lds_char;

template <int D>
__device__ __forceinline__ int lds_off_tree(int row, int chunk) {
    if constexpr (D == 128) return lds_off128(row, chunk);
    else return lds_off64(row, chunk);
}

#define LV_TREE_UNUSED (-2)   // parents[] entry of a slot that holds no token

__device__ __forceinline__ int tree_len(const TreeParams& p, int s) {
    const int len = p.cache_lens[s];
    return min(max(len, 0), p.rows - p.n);   // never outside the cache, whatever the caller's array says
}
__device__ __forceinline__ int tree_tiles(const TreeParams& p, int s) { return (tree_len(p, s) + p.n + LV_TREE_TILE - 1) / LV_TREE_TILE; }

// cum[s] = tiles of sequences 0 .. s (one wave); returns after a barrier of the whole workgroup
__device__ __forceinline__ void tree_scan(const TreeParams& p, int* cum) {
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int carry = 0;
        for (int s0 = 0; s0 < p.batch; s0 += 64) {
            int x = s0 + lane < p.batch ? tree_tiles(p, s0 + lane) : 0;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int y = __shfl_up(x, off);
                if (lane >= off) x += y;
            }
            if (s0 + lane < p.batch) cum[s0 + lane] = carry + x;
            carry += __shfl(x, 63);
        }
    }
    __syncthreads();
}

template <int D, int WR, int MOD>
__global__ __launch_bounds__(256, 2) void lv_tree_kernel(TreeParams p) {
    constexpr int BN = LV_TREE_TILE;
    constexpr int WK = 4 / WR;            // waves side by side over the keys
    constexpr int KPW = BN / WK;          // keys of a tile per wave
    constexpr int KS = D / 16;
    constexpr int MT = D / 32;
    constexpr int ROWB = D * 2;
    constexpr int TILEB = BN * ROWB;
    constexpr int CPR = D / 8;
    constexpr int NT = 256;
    constexpr int NLD = (BN * CPR) / NT;
    constexpr float RESCALE_LOG2 = 8.0f;

    extern __shared__ __attribute__((aligned(16))) char smem[];
    lds_char* const ldsK = (lds_char*)smem;
    lds_char* const ldsV = ldsK + TILEB;
    int* const cum = reinterpret_cast<int*>(smem + 2 * TILEB);          // [LV_TREE_MAX_BATCH]
    int* const par = cum + LV_TREE_MAX_BATCH;                           // [LV_TREE_MAX_TOKENS]
    int* const depth = par + LV_TREE_MAX_TOKENS;                        // [LV_TREE_MAX_TOKENS]
    uint32_t* const anc = reinterpret_cast<uint32_t*>(depth + LV_TREE_MAX_TOKENS);   // [tokens][words]: ancestors of a token
    float* const stat = reinterpret_cast<float*>(anc + LV_TREE_MAX_TOKENS * (LV_TREE_MAX_TOKENS / 32));   // [2][4][32]

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

    tree_scan(p, cum);
    const int64_t total = cum[p.batch - 1];
    const int64_t G = min((int64_t)p.shares, total);
    if (g >= G) return;
    int64_t tile = g * total / G;
    const int64_t tile_end = (g + 1) * total / G;
    int s = 0;
    while (cum[s] <= tile) ++s;

    const int64_t k_tile = (int64_t)BN * p.k_rs, v_tile = (int64_t)BN * p.v_rs;
    // thread -> 16-byte chunk tid % CPR of rows tid / CPR + RSTEP i (RSTEP is a period of the LDS swizzle)
    constexpr int RSTEP = NT / CPR;
    static_assert(RSTEP % 16 == 0, "the swizzle repeats every 16 rows");
    const int st_lds = lds_off_tree<D>(tid / CPR, tid % CPR);
    const int st_koff = (int)(tid / CPR * p.k_rs * 2) + tid % CPR * 16, st_voff = (int)(tid / CPR * p.v_rs * 2) + tid % CPR * 16;
    const int k_step = (int)(RSTEP * p.k_rs * 2), v_step = (int)(RSTEP * p.v_rs * 2);
    u32x4 kreg[NLD], vreg[NLD];
    auto issue_loads = [&](int sq, int t) __attribute__((always_inline)) {
        const int rows = min(tree_len(p, sq) + p.n - t * BN, BN);       // >= 1: the tile is one of the sequence's
        // rows past the sequence's last key read as zero (buffer bounds check) and are masked below
        auto krs = __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(p.k + (int64_t)sq * p.k_bs + (int64_t)kvh * p.k_hs + t * k_tile), 0,
                                                     (uint32_t)((rows - 1) * p.k_rs * 2 + ROWB), 0x00020000);
        auto vrs = __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(p.v + (int64_t)sq * p.v_bs + (int64_t)kvh * p.v_hs + t * v_tile), 0,
                                                     (uint32_t)((rows - 1) * p.v_rs * 2 + ROWB), 0x00020000);
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            kreg[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(krs, st_koff + i * k_step, 0, 0));
            vreg[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vrs, st_voff + i * v_step, 0, 0));
        }
    };

    lds_char* k_ptr[KS];   // K row read: row r of the 32-key sub-tile, chunk 2ks + h
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k_ptr[ks] = ldsK + lds_off_tree<D>(KPW * wk + r, 2 * ks + h);
    const int i16 = lane & 15, q4 = i16 >> 2, p4 = i16 & 3, gl = (lane >> 4) & 1;
    lds_char* v_ptr[MT][2];   // V transposed read
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int jh = 0; jh < 2; ++jh)
            v_ptr[mt][jh] = ldsV + lds_off_tree<D>(8 * jh + 4 * h + q4, 4 * mt + 2 * gl + (p4 >> 1)) + 8 * (p4 & 1) + KPW * wk * ROWB;

    // this lane's query row: row -> (token, head of the group)
    const int row = 32 * (WR * rb + wr) + r;
    const int n_rows = p.n * p.group;
    const int rowc = min(row, n_rows - 1);
    const int token = rowc / p.group, head = kvh * p.group + rowc % p.group;
    float nslope2 = 0.f;
    if constexpr ((MOD & LV_SCORE_BIAS) != 0) nslope2 = -1.4426950408889634f * p.score.slopes[head];
    const float c = MOD != 0 ? 1.f : p.scale_log2e;

    issue_loads(s, (int)(tile - (s ? cum[s - 1] : 0)));

    while (tile < tile_end) {
        // ---------------- one sequence of this share ----------------
        const int len = tree_len(p, s), keys = len + p.n;
        const int t0 = (int)(tile - (s ? cum[s - 1] : 0));
        const int t1 = (int)(min(tile_end, (int64_t)cum[s]) - (s ? cum[s - 1] : 0));
        const bool sees_tree = t1 * BN > len;

        bf16x8 qf[KS];
        const __bf16* qptr = p.q + (int64_t)s * p.q_bs + (int64_t)token * p.q_ns + (int64_t)head * p.q_hs + 8 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(qptr + 16 * ks);

        int my_depth = token;             // without parents the tokens are a chain
        bool unused = false;
        if (p.parents) {
            const int* pp = p.parents + (int64_t)s * p.parents_bs;
            __syncthreads();              // the previous sequence's arrays are no longer read
            for (int i = tid; i < p.n; i += NT) {
                const int x = pp[i];
                par[i] = x < i ? x : -1;  // a parent stands before its child: the walk below always ends
            }
            __syncthreads();
            for (int i = tid; i < p.n; i += NT) {
                if (sees_tree)
                    for (int x = 0; x < words; ++x) anc[i * words + x] = 0;
                int dep = -1, at = i;
                if (par[i] != LV_TREE_UNUSED)
                    while (at >= 0) {
                        if (sees_tree) anc[i * words + (at >> 5)] |= 1u << (at & 31);
                        ++dep;
                        at = par[at];
                    }
                depth[i] = max(dep, 0);
            }
            __syncthreads();
            my_depth = depth[token];
            unused = par[token] == LV_TREE_UNUSED;
        }
        const bool live = row < n_rows && !unused;

        f32x16 oacc[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 16; ++i) oacc[mt][i] = 0.f;
        float m_run = -1e30f, l_run = 0.f;

        for (int t = t0; t < t1; ++t) {
            const bool tree_tile = (t + 1) * BN > len;     // holds drafted keys, or keys past the end
            if (tree_tile && p.parents) {
                // rows of unused slots hold whatever was there: zero, so that not even a NaN gets through P = 0
#pragma unroll
                for (int i = 0; i < NLD; ++i) {
                    const int j = t * BN + (tid + NT * i) / CPR - len;
                    if (j >= 0 && j < p.n && par[j] == LV_TREE_UNUSED) { kreg[i] = u32x4{0, 0, 0, 0}; vreg[i] = u32x4{0, 0, 0, 0}; }
                }
            }
#pragma unroll
            for (int i = 0; i < NLD; ++i) {      // (waits for tile t's loads)
                *(LDS_PTR(u32x4, ldsK + st_lds + i * RSTEP * ROWB)) = kreg[i];
                *(LDS_PTR(u32x4, ldsV + st_lds + i * RSTEP * ROWB)) = vreg[i];
            }
            __syncthreads();
            ++tile;
            if (tile < tile_end) issue_loads(t + 1 < t1 ? s : s + 1, t + 1 < t1 ? t + 1 : 0);
#pragma unroll 1
            for (int sub = 0; sub < KPW / 32; ++sub) {
                const int kb0 = t * BN + KPW * wk + 32 * sub;
                if (kb0 >= keys) break;
                const int soff = 32 * sub * ROWB;
                f32x16 x;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const bf16x8 kf = *(LDS_PTR(bf16x8, k_ptr[ks] + soff));
                    x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ks], x, 0, 0, 0);
                }
                const bool masked = kb0 + 32 > len;
                if constexpr (MOD != 0) {
                    const int jl = kb0 + 4 * h;
                    const float fq = (float)(len + my_depth - jl);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float dist = fq - (float)((i & 3) + 8 * (i >> 2));
                        if constexpr ((MOD & LV_SCORE_BIAS) != 0)
                            if (masked && p.parents) {       // a drafted key stands at its depth, not at its row
                                const int j = jl + (i & 3) + 8 * (i >> 2) - len;
                                if (j >= 0) dist = (float)(my_depth - depth[min(j, p.n - 1)]);
                            }
                        x[i] = lv_score<MOD>(x[i], p.scale_log2e, p.score, nslope2, dist);
                    }
                }
                if (masked) {
                    // bit e of `vis`: key kb0 + e visible to this lane's token
                    uint32_t vis;
                    const int j0 = kb0 - len;          // first key of the sub-tile, counted from the first drafted one
                    if (p.parents) {
                        const uint32_t* aw = anc + token * words;
                        const int lo = j0 >> 5;        // (arithmetic shift: -1 for a sub-tile that starts in the cache)
                        const uint32_t a = lo < 0 ? 0xffffffffu : (lo < words ? aw[lo] : 0u);
                        const uint32_t b = lo + 1 < words ? aw[lo + 1] : 0u;
                        vis = (uint32_t)((((uint64_t)b << 32) | a) >> (j0 & 31));
                    } else {
                        const int last = token - j0;   // keys up to the token's own
                        vis = last >= 31 ? 0xffffffffu : (last < 0 ? 0u : (2u << last) - 1u);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int e = (i & 3) + 8 * (i >> 2) + 4 * h;
                        x[i] = (vis >> e) & 1 ? x[i] : -INFINITY;
                    }
                }
                float mx = x[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
                mx = pair32_max(mx);
                const float m_new = fmaxf(m_run, mx);
                const bool grow = (m_new - m_run) * c > RESCALE_LOG2;
                if (__any(grow)) {
                    const float alpha = fast_exp2((m_run - m_new) * c);
                    m_run = m_new;
                    l_run *= alpha;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 16; ++i) oacc[mt][i] *= alpha;
                }
                const float mc = m_run * c;
                float rs = 0.f;
                bf16x8 pf[2];     // P rounds to bf16, the matrix pipe's type; its sum is taken before the rounding
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float pv = fast_exp2(__builtin_fmaf(x[i], c, -mc));
                    rs += pv;
                    pf[i >> 3][i & 7] = (__bf16)pv;
                }
                l_run += rs;
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    const int voff = soff + 16 * s2 * ROWB;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, v_ptr[mt][0] + voff));
                        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, v_ptr[mt][1] + voff));
                        bf16x8 vf;
                        vf[0] = lo[0]; vf[1] = lo[1]; vf[2] = lo[2]; vf[3] = lo[3];
                        vf[4] = hi[0]; vf[5] = hi[1]; vf[6] = hi[2]; vf[7] = hi[3];
                        oacc[mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[s2], oacc[mt], 0, 0, 0);
                    }
                }
            }
            __syncthreads();        // every wave is done with the tile before it is overwritten
        }

        // ---------------- this share's result for the sequence -> partial slot g + s ----------------
        const int64_t part = ((int64_t)(kvh * p.n_rb + rb) * p.slots + g + s) * (32 * WR) + 32 * wr;   // first row of this wave's block
        const float unit2 = MOD != 0 ? 0.6931471805599453f : p.scale;
        const float l_w = pair32_sum(l_run);
        if constexpr (WK == 1) {
            const float inv = (l_w > 0.f && live) ? 1.f / l_w : 0.f;
            float* po = p.part_o + (part + r) * D + 4 * h;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4)
                    *reinterpret_cast<f32x4*>(po + 32 * mt + 8 * g4) =
                        f32x4{oacc[mt][4 * g4] * inv, oacc[mt][4 * g4 + 1] * inv, oacc[mt][4 * g4 + 2] * inv, oacc[mt][4 * g4 + 3] * inv};
            if (h == 0) p.part_lse[part + r] = (l_w > 0.f && live) ? m_run * unit2 + __logf(l_w) : -INFINITY;
        } else {
            if (h == 0) {
                stat[w * 32 + r] = m_run;
                stat[128 + w * 32 + r] = l_w;
            }
            __syncthreads();
            float m_tot = -1e30f;
#pragma unroll
            for (int i = 0; i < WK; ++i) m_tot = fmaxf(m_tot, stat[(i * WR + wr) * 32 + r]);
            float l_tot = 0.f;
#pragma unroll
            for (int i = 0; i < WK; ++i) l_tot += stat[128 + (i * WR + wr) * 32 + r] * fast_exp2((stat[(i * WR + wr) * 32 + r] - m_tot) * c);
            const float sc = fast_exp2((m_run - m_tot) * c);
            float* const obuf = reinterpret_cast<float*>(smem);           // the (free) tile memory: [4 waves][MT][64 lanes][16]
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float* dst = obuf + ((w * MT + mt) * 64 + lane) * 16;
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4)
                    *reinterpret_cast<f32x4*>(dst + 4 * g4) = f32x4{oacc[mt][4 * g4] * sc, oacc[mt][4 * g4 + 1] * sc,
                                                                     oacc[mt][4 * g4 + 2] * sc, oacc[mt][4 * g4 + 3] * sc};
            }
            __syncthreads();
            const float inv = (l_tot > 0.f && live) ? 1.f / l_tot : 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                if (mt % WK != wk) continue;       // the key waves of a row block share out its d columns
                f32x4 acc[4];
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) acc[g4] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < WK; ++i) {
                    const float* src = obuf + (((i * WR + wr) * MT + mt) * 64 + lane) * 16;
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) acc[g4] += *reinterpret_cast<const f32x4*>(src + 4 * g4);
                }
                float* po = p.part_o + (part + r) * D + 32 * mt + 4 * h;
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) *reinterpret_cast<f32x4*>(po + 8 * g4) = acc[g4] * inv;
            }
            if (wk == 0 && h == 0) p.part_lse[part + r] = (l_tot > 0.f && live) ? m_tot * unit2 + __logf(l_tot) : -INFINITY;
            __syncthreads();        // the next tile goes where obuf is
        }
        ++s;
    }
}

// out / lse of a row = the log-sum-exp merge of its sequence's slots, in order.  Eight rows per workgroup, 32 threads per row.
template <int D>
__global__ __launch_bounds__(256) void lv_tree_join_kernel(TreeParams p, int rows_pb) {
    __shared__ int cum[LV_TREE_MAX_BATCH];
    tree_scan(p, cum);
    const int64_t total = cum[p.batch - 1];
    const int64_t G = min((int64_t)p.shares, total);
    const int64_t idx = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;       // (sequence, KV head, row)
    const int n_rows = p.n * p.group;
    if (idx >= (int64_t)p.batch * p.hkv * n_rows) return;
    const int row = (int)(idx % n_rows), kvh = (int)(idx / n_rows % p.hkv), s = (int)(idx / n_rows / p.hkv);
    const int64_t first = s ? cum[s - 1] : 0, last = cum[s] - 1;
    // share that holds tile t: the largest g with floor(g total / G) <= t
    const int64_t g0 = ((first + 1) * G - 1) / total, g1 = ((last + 1) * G - 1) / total;
    const int rb = row / rows_pb;
    const int64_t part = ((int64_t)(kvh * p.n_rb + rb) * p.slots + g0 + s) * rows_pb + row % rows_pb;
    const int np = (int)(g1 - g0 + 1);
    const float* lp = p.part_lse + part;
    float m = -INFINITY;
    for (int i = 0; i < np; ++i) m = fmaxf(m, lp[(int64_t)i * rows_pb]);
    constexpr int C = D / 32;                 // columns per thread
    const int col = (threadIdx.x & 31) * C;
    float acc[C], tot = 0.f;
#pragma unroll
    for (int e = 0; e < C; ++e) acc[e] = 0.f;
    if (m > -INFINITY) {
        const float* po = p.part_o + part * D + col;
#pragma unroll 4
        for (int i = 0; i < np; ++i) {
            const float wgt = __expf(lp[(int64_t)i * rows_pb] - m);
            tot += wgt;
#pragma unroll
            for (int e = 0; e < C; ++e) acc[e] += wgt * po[(int64_t)i * rows_pb * D + e];
        }
    }
    const float inv = tot > 0.f ? 1.f / tot : 0.f;
    const int token = row / p.group, head = kvh * p.group + row % p.group;
    __bf16* op = p.o + (int64_t)s * p.o_bs + (int64_t)token * p.o_ns + (int64_t)head * p.o_hs + col;
#pragma unroll
    for (int e = 0; e < C; ++e) op[e] = (__bf16)(acc[e] * inv);
    if (p.lse && (threadIdx.x & 31) == 0) p.lse[((int64_t)s * p.n + token) * p.hq + head] = tot > 0.f ? m + __logf(tot) : -INFINITY;
}

// query rows per workgroup: 32, 64 or 128.  Up to 32 rows all four waves split the keys; from 65 on none do
static int tree_rows_per_block(int n_rows) { return n_rows <= 32 ? 32 : (n_rows <= 64 ? 64 : 128); }

struct TreePlan { int rows_pb, n_rb, shares, slots; int64_t part_rows; };
// Shares per KV head: two workgroups fit a compute unit, so 512 workgroups fill the chip once; never more shares than tiles.
static TreePlan tree_plan(int batch, int n, int rows, int hq, int hkv) {
    TreePlan t;
    const int n_rows = n * (hq / hkv);
    t.rows_pb = tree_rows_per_block(n_rows);
    t.n_rb = (n_rows + t.rows_pb - 1) / t.rows_pb;
    const int64_t tiles = (int64_t)batch * ((rows + LV_TREE_TILE - 1) / LV_TREE_TILE);
    int64_t g = (512 + (int64_t)hkv * t.n_rb - 1) / ((int64_t)hkv * t.n_rb);
    if (g > tiles) g = tiles;
    t.shares = (int)g;
    t.slots = (int)g + batch - 1;
    t.part_rows = (int64_t)hkv * t.n_rb * t.slots * t.rows_pb;
    return t;
}

template <int D, int WR>
static void launch_tree(const TreeParams& p, int mod, dim3 grid, hipStream_t stream) {
    const size_t lds = (size_t)2 * LV_TREE_TILE * D * 2 + LV_TREE_MAX_BATCH * 4 + LV_TREE_MAX_TOKENS * 8 +
                       LV_TREE_MAX_TOKENS * (LV_TREE_MAX_TOKENS / 32) * 4 + 1024;
    // (D = 64: the join buffer of the epilogue, 4 waves x 2 x 4 KB, is as large as the two tiles)
    switch (mod) {
        case 0: hipLaunchKernelGGL((lv_tree_kernel<D, WR, 0>), grid, dim3(256), lds, stream, p); break;
        case LV_SCORE_CAP: hipLaunchKernelGGL((lv_tree_kernel<D, WR, LV_SCORE_CAP>), grid, dim3(256), lds, stream, p); break;
        case LV_SCORE_BIAS: hipLaunchKernelGGL((lv_tree_kernel<D, WR, LV_SCORE_BIAS>), grid, dim3(256), lds, stream, p); break;
        default: hipLaunchKernelGGL((lv_tree_kernel<D, WR, LV_SCORE_CAP | LV_SCORE_BIAS>), grid, dim3(256), lds, stream, p);
    }
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
    if (!(softmax_scale > -1e30f && softmax_scale < 1e30f)) return lv_fail(LV_EINVAL, "lvattn_tree: softmax_scale is not finite");
    const TreePlan t = tree_plan(batch, n, rows, hq, hkv);
    const int64_t need = t.part_rows * (d + 1) * (int64_t)sizeof(float);
    if (workspace_bytes < need) return lv_fail(LV_ESIZE, "lvattn_tree: %lld bytes of workspace needed, room for %lld", (long long)need, (long long)workspace_bytes);
    const int64_t units = (int64_t)hkv * t.shares, blocks = (units + 7) / 8 * 8 * t.n_rb;
    const int64_t join = ((int64_t)batch * hkv * n * (hq / hkv) + 7) / 8;
    if (blocks > 0x7fffffffLL || join > 0x7fffffffLL) return lv_fail(LV_EINVAL, "lvattn_tree: grid too large");
    TreeParams p{};
    p.q = (const __bf16*)q; p.k = (const __bf16*)k; p.v = (const __bf16*)v; p.o = (__bf16*)out; p.lse = lse;
    p.cache_lens = cache_lens; p.parents = parents; p.parents_bs = parents_batch_stride;
    p.part_o = (float*)workspace; p.part_lse = p.part_o + t.part_rows * d;
    p.batch = batch; p.n = n; p.rows = rows; p.hq = hq; p.hkv = hkv; p.group = hq / hkv;
    p.n_rb = t.n_rb; p.shares = t.shares; p.slots = t.slots;
    p.q_bs = q_bs; p.q_ns = q_ns; p.q_hs = q_hs; p.k_bs = k_bs; p.k_rs = k_rs; p.k_hs = k_hs; p.v_bs = v_bs; p.v_rs = v_rs; p.v_hs = v_hs;
    p.o_bs = o_bs; p.o_ns = o_ns; p.o_hs = o_hs;
    p.scale = softmax_scale; p.scale_log2e = softmax_scale * 1.4426950408889634f;
    p.score = lv_score_rule(softmax_scale, softcap, slopes);
    const int mod = lv_score_mod(softcap, slopes) & (LV_SCORE_CAP | LV_SCORE_BIAS);
    const dim3 grid((unsigned)blocks);
    if (d == 128) {
        if (t.rows_pb == 32) launch_tree<128, 1>(p, mod, grid, (hipStream_t)stream);
        else if (t.rows_pb == 64) launch_tree<128, 2>(p, mod, grid, (hipStream_t)stream);
        else launch_tree<128, 4>(p, mod, grid, (hipStream_t)stream);
    } else {
        if (t.rows_pb == 32) launch_tree<64, 1>(p, mod, grid, (hipStream_t)stream);
        else if (t.rows_pb == 64) launch_tree<64, 2>(p, mod, grid, (hipStream_t)stream);
        else launch_tree<64, 4>(p, mod, grid, (hipStream_t)stream);
    }
    if (hipGetLastError() != hipSuccess) return lv_fail(LV_ELAUNCH, "lvattn_tree: launch failed");
    if (d == 128) hipLaunchKernelGGL((lv_tree_join_kernel<128>), dim3((unsigned)join), dim3(256), 0, (hipStream_t)stream, p, t.rows_pb);
    else hipLaunchKernelGGL((lv_tree_join_kernel<64>), dim3((unsigned)join), dim3(256), 0, (hipStream_t)stream, p, t.rows_pb);
    return hipGetLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "lvattn_tree: launch failed");
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

extern "C" int lv_tree_accept(void* k, void* v, float* weight, const int32_t* cache_lens, const int32_t* path, const int32_t* n_accept, int batch,
                              int n, int rows, int hkv, int d, int64_t k_bs, int64_t k_rs, int64_t k_hs, int64_t v_bs, int64_t v_rs, int64_t v_hs,
                              int64_t w_bs, int64_t w_hs, void* stream) {
    if (!k || !v || !cache_lens || !path || !n_accept) return lv_fail(LV_EINVAL, "lv_tree_accept: null pointer");
    if (d != 64 && d != 128) return lv_fail(LV_EINVAL, "lv_tree_accept: head dim %d (64 or 128)", d);
    if (batch <= 0 || hkv <= 0 || n <= 0 || rows < n) return lv_fail(LV_EINVAL, "lv_tree_accept: bad sizes");
    if ((((uintptr_t)k | (uintptr_t)v) & 15) || ((k_bs | k_rs | k_hs | v_bs | v_rs | v_hs) & 7))
        return lv_fail(LV_EINVAL, "lv_tree_accept: k / v must be 16-byte aligned with strides %% 8 == 0");
    if ((int64_t)batch * hkv > 0x7fffffffLL) return lv_fail(LV_EINVAL, "lv_tree_accept: grid too large");
    AcceptParams p{};
    p.k = (__bf16*)k; p.v = (__bf16*)v; p.weight = weight; p.cache_lens = cache_lens; p.path = path; p.n_accept = n_accept;
    p.n = n; p.rows = rows; p.hkv = hkv; p.d = d;
    p.k_bs = k_bs; p.k_rs = k_rs; p.k_hs = k_hs; p.v_bs = v_bs; p.v_rs = v_rs; p.v_hs = v_hs; p.w_bs = w_bs; p.w_hs = w_hs;
    hipLaunchKernelGGL(lv_tree_accept_kernel, dim3((unsigned)(batch * hkv)), dim3(512), 0, (hipStream_t)stream, p);
    return hipGetLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "lv_tree_accept: launch failed");
}
