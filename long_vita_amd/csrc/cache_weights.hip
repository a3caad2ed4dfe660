// Attention weight received by every cached key, for gfx950: what cache eviction goes by.
//
//   w_out[kvh, j] = w_in[kvh, j] + sum over tokens i and query heads h of kvh's group of rho_i exp(t_ij - lse_ih)
//
// t and the visible keys are those of attn_tree.hip, lse comes from the attention itself, rho is an optional weight per token
// (0 for drafted tokens that were not accepted).  One product, S = Q K^T, with the KEY on the lane (32x32x16 MFMA, A = query
// rows from LDS, B = keys): a wave keeps the fragments of its 64 keys in registers for the whole kernel, so K is read once,
// and a key's sum over a tile of query rows is a sum over its lane's 16 accumulators.  Nothing is ever summed by atomics.
//
// A workgroup is 4 waves: 4 / RW over keys, RW over alternate tiles of 32 query rows (few rows: one tile, all waves on keys;
// a whole prompt's rows: two).  When there are fewer key blocks than the chip has room for, the rows are cut into pieces
// whose sums go to a workspace and are added in order.  Few rows: bound by K's bytes.  Many: 8 MFMAs (256 cycles) against 16
// exponentials, multiply-adds and adds per 32 x 32 scores, so the vector work bounds it.
#include "internal.h"
#include "../../include/lvattn.h"

typedef __attribute__((address_space(3))) char lds_char;

template <int D>
__device__ __forceinline__ int lds_off_w(int row, int chunk) {
    if constexpr (D == 128) return lds_off128(row, chunk);
    else return lds_off64(row, chunk);
}

template <int D, int MOD, int RW>
__global__ __launch_bounds__(256, 2) void lv_key_weights_kernel(WeightParams p) {
    constexpr int KWAVES = 4 / RW;
    constexpr int KB = 64 * KWAVES;       // keys per workgroup
    constexpr int KS = D / 16;
    constexpr int CPR = D / 8;
    constexpr int ROWB = D * 2;
    constexpr int TR = 32 * RW;           // query rows per step
    constexpr int NLD = TR * CPR / 256;   // 16-byte chunks per thread and step
    static_assert(TR * CPR % 256 == 0, "whole chunks per thread");

    __shared__ __attribute__((aligned(16))) char qbuf[2][TR * ROWB];
    __shared__ __attribute__((aligned(16))) float cst[2][TR];     // log2(rho) - lse log2(e); -inf: the row counts for nothing
    __shared__ __attribute__((aligned(16))) float rpos[2][TR];    // position of the row's token, counted from the cache's start
    __shared__ __attribute__((aligned(16))) float rslope[2][TR];  // -log2(e) slope of the row's head
    __shared__ int rtok[2][TR];
    __shared__ float red[RW > 1 ? (RW - 1) * KB : 1];
    __shared__ int par[LV_TREE_MAX_TOKENS], depth[LV_TREE_MAX_TOKENS];
    __shared__ uint32_t anc[LV_TREE_MAX_TOKENS * (LV_TREE_MAX_TOKENS / 32)];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kw = w % KWAVES, rw = w / KWAVES;
    const int r = lane & 31, h = lane >> 5;

    // heads and sequences fastest, then row pieces, then key blocks from the first (under a causal rule the heaviest) on
    const int bh = blockIdx.x % (p.batch * p.hkv);
    const int rest = blockIdx.x / (p.batch * p.hkv);
    const int piece = rest % p.pieces, kb = rest / p.pieces;
    const int s = bh / p.hkv, kvh = bh % p.hkv;
    const int len = min(max(p.cache_lens[s], 0), p.rows - p.n), keys = len + p.n;
    const int k0 = kb * KB;
    const int64_t w_in0 = (int64_t)s * p.wi_bs + (int64_t)kvh * p.wi_hs, w_out0 = (int64_t)s * p.wo_bs + (int64_t)kvh * p.wo_hs;
    if (k0 >= keys) {                     // behind the last key: the weights stay as they are
        if (piece == 0 && p.w_in != p.w_out)
            for (int j = k0 + tid; j < min(k0 + KB, p.rows); j += 256) p.w_out[w_out0 + j] = p.w_in[w_in0 + j];
        return;
    }
    const int n_rows = p.n * p.group;
    const int words = (p.n + 31) >> 5;

    if (p.parents) {
        const int* pp = p.parents + (int64_t)s * p.parents_bs;
        for (int i = tid; i < p.n; i += 256) {
            const int x = pp[i];
            par[i] = x < i ? x : -1;      // a parent stands before its child: the walk below always ends
        }
        __syncthreads();
        const bool sees_tree = k0 + KB > len;
        if (sees_tree || (MOD & LV_SCORE_BIAS) != 0) {
            for (int i = tid; i < p.n; i += 256) {
                for (int x = 0; x < words; ++x) anc[i * words + x] = 0;
                int dep = -1, at = i;
                if (par[i] != -2)
                    while (at >= 0) {
                        anc[i * words + (at >> 5)] |= 1u << (at & 31);
                        ++dep;
                        at = par[at];
                    }
                depth[i] = max(dep, 0);
            }
            __syncthreads();
        }
    }

    // ---- this wave's keys: two groups of 32, fragments for the whole kernel
    bf16x8 kf[2][KS];
    int key[2];
    float kpos[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int base = k0 + 64 * kw + 32 * g;
        key[g] = base + r;
        const int valid = min(max(keys - base, 0), 32);      // rows past the last key read as zero and count for nothing
        auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<__bf16*>(p.k + (int64_t)s * p.k_bs + (int64_t)kvh * p.k_hs + (int64_t)base * p.k_rs), 0,
                                                    valid ? (uint32_t)((valid - 1) * p.k_rs * 2 + ROWB) : 0u, 0x00020000);
        const int off = (int)(r * p.k_rs * 2) + 16 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kf[g][ks] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, off + 32 * ks, 0, 0));
        kpos[g] = (float)key[g];
        if constexpr ((MOD & LV_SCORE_BIAS) != 0)
            if (p.parents && key[g] >= len && key[g] < keys) kpos[g] = (float)(len + depth[key[g] - len]);
    }

    // ---- the rows that see any key of the block, this piece's share of them
    int row_lo = 0;
    if (!p.parents && k0 > len) row_lo = (k0 - len) * p.group / TR * TR;     // a chain: drafted key j is seen from token j on
    const int steps = (n_rows - row_lo + TR - 1) / TR;
    const int st0 = (int)((int64_t)steps * piece / p.pieces), st1 = (int)((int64_t)steps * (piece + 1) / p.pieces);

    u32x4 qreg[NLD];
    float creg = -INFINITY, preg = 0.f, sreg = 0.f;
    int treg = 0;
    auto load_step = [&](int st) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            const int cidx = tid + 256 * i;
            const int row = row_lo + st * TR + cidx / CPR;
            qreg[i] = u32x4{0, 0, 0, 0};          // rows that count for nothing are zero: whatever they hold cannot reach a sum
            if (row < n_rows) {
                const int token = row / p.group, head = kvh * p.group + row % p.group;
                const bool on = (!p.row_weight || p.row_weight[(int64_t)s * p.n + token] > 0.f) && !(p.parents && par[token] == -2);
                if (on) qreg[i] = *reinterpret_cast<const u32x4*>(p.q + (int64_t)s * p.q_bs + (int64_t)token * p.q_ns + (int64_t)head * p.q_hs + cidx % CPR * 8);
            }
        }
        if (tid < TR) {
            const int row = row_lo + st * TR + tid;
            creg = -INFINITY;
            if (row < n_rows) {
                const int token = row / p.group, head = kvh * p.group + row % p.group;
                const float rho = p.row_weight ? p.row_weight[(int64_t)s * p.n + token] : 1.f;
                const float l = p.lse[((int64_t)s * p.n + token) * p.hq + head];
                treg = token;
                if (rho > 0.f && l > -INFINITY && !(p.parents && par[token] == -2))
                    creg = (p.row_weight ? __builtin_amdgcn_logf(rho) : 0.f) - l * 1.4426950408889634f;
                if constexpr ((MOD & LV_SCORE_BIAS) != 0) {
                    preg = (float)(len + (p.parents ? depth[token] : token));
                    sreg = -1.4426950408889634f * p.score.slopes[head];
                }
            }
        }
    };
    auto write_step = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            const int cidx = tid + 256 * i;
            *reinterpret_cast<u32x4*>(qbuf[buf] + lds_off_w<D>(cidx / CPR, cidx % CPR)) = qreg[i];
        }
        if (tid < TR) {
            cst[buf][tid] = creg;
            rtok[buf][tid] = treg;
            if constexpr ((MOD & LV_SCORE_BIAS) != 0) { rpos[buf][tid] = preg; rslope[buf][tid] = sreg; }
        }
    };

    float sum[2] = {0.f, 0.f}, lost[2] = {0.f, 0.f};     // a key may collect tens of thousands of terms: compensated sums
    if (st0 < st1) {
        load_step(st0);
        write_step(0);
    }
    __syncthreads();
    for (int st = st0; st < st1; ++st) {
        const int buf = (st - st0) & 1;
        if (st + 1 < st1) load_step(st + 1);
        const int row0 = row_lo + st * TR + 32 * rw;      // first row of this wave's tile
        if (row0 < n_rows) {
            f32x4 cv[4];
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) cv[q4] = *reinterpret_cast<const f32x4*>(&cst[buf][32 * rw + 8 * q4 + 4 * h]);
            f32x16 x[2];
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[g][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const bf16x8 qf = *(LDS_PTR(bf16x8, (lds_char*)qbuf[buf] + lds_off_w<D>(32 * rw + r, 2 * ks + h)));
                x[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf, kf[0][ks], x[0], 0, 0, 0);
                x[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf, kf[1][ks], x[1], 0, 0, 0);
            }
            // smallest token of the tile against the last key of the wave: every row sees every key?
            const int first_token = row0 / p.group;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int kl = k0 + 64 * kw + 32 * g + 31;            // last key of the group
                const bool masked = kl >= keys || (kl >= len && (p.parents || kl - len > first_token));
                const int jt = key[g] - len;
                float pv[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int rr = 32 * rw + (i & 3) + 8 * (i >> 2) + 4 * h;
                    float t;
                    if constexpr (MOD != 0) {
                        float dist = 0.f, sl = 0.f;
                        if constexpr ((MOD & LV_SCORE_BIAS) != 0) { dist = rpos[buf][rr] - kpos[g]; sl = rslope[buf][rr]; }
                        t = lv_score<MOD>(x[g][i], p.scale_log2e, p.score, sl, dist) + cv[i >> 2][i & 3];
                    } else {
                        t = __builtin_fmaf(x[g][i], p.scale_log2e, cv[i >> 2][i & 3]);
                    }
                    pv[i] = fast_exp2(t);
                }
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int rr = 32 * rw + (i & 3) + 8 * (i >> 2) + 4 * h;
                        bool vis = key[g] < keys;
                        if (jt >= 0 && vis) {
                            const int token = rtok[buf][rr];
                            vis = p.parents ? (anc[token * words + (jt >> 5)] >> (jt & 31)) & 1 : jt <= token;
                        }
                        pv[i] = vis ? pv[i] : 0.f;
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
        if (st + 1 < st1) write_step(buf ^ 1);     // (that buffer's last readers passed the barrier below a step ago)
        __syncthreads();
    }

    float tot[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) tot[g] = pair32_sum(sum[g] - lost[g]);
    if constexpr (RW > 1) {
        if (rw > 0 && h == 0)
#pragma unroll
            for (int g = 0; g < 2; ++g) red[(rw - 1) * KB + 64 * kw + 32 * g + r] = tot[g];
        __syncthreads();
        if (rw == 0)
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int x = 0; x < RW - 1; ++x) tot[g] += red[x * KB + 64 * kw + 32 * g + r];
    }
    if (rw == 0 && h == 0) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if (key[g] >= p.rows) continue;
            if (p.pieces > 1) {
                if (key[g] < keys) p.part[((int64_t)piece * p.batch * p.hkv + bh) * p.rows + key[g]] = tot[g];
            } else {
                p.w_out[w_out0 + key[g]] = p.w_in[w_in0 + key[g]] + (key[g] < keys ? tot[g] : 0.f);
            }
        }
    }
}

// w_out = w_in + the pieces' sums, first piece first
__global__ __launch_bounds__(256) void lv_key_weights_join_kernel(WeightParams p, int key_block) {
    const int bh = blockIdx.y;
    const int s = bh / p.hkv, kvh = bh % p.hkv;
    const int j = blockIdx.x * 256 + threadIdx.x;
    const int keys = min(max(p.cache_lens[s], 0), p.rows - p.n) + p.n;
    // blocks that begin behind the last key were copied by the first kernel
    if (j >= p.rows || j / key_block * key_block >= keys) return;
    float x = p.w_in[(int64_t)s * p.wi_bs + (int64_t)kvh * p.wi_hs + j];
    if (j < keys) {
        float add = 0.f;
        for (int i = 0; i < p.pieces; ++i) add += p.part[((int64_t)i * p.batch * p.hkv + bh) * p.rows + j];
        x += add;
    }
    p.w_out[(int64_t)s * p.wo_bs + (int64_t)kvh * p.wo_hs + j] = x;
}

struct WeightPlan { int rw, key_block, key_blocks, pieces; };
static WeightPlan weight_plan(int batch, int n, int rows, int hq, int hkv) {
    WeightPlan t;
    const int n_rows = n * (hq / hkv);
    t.rw = n_rows <= 32 ? 1 : 2;
    t.key_block = 64 * (4 / t.rw);
    t.key_blocks = (rows + t.key_block - 1) / t.key_block;
    const int64_t units = (int64_t)batch * hkv * t.key_blocks;
    // two workgroups fit a compute unit; a piece keeps at least 8 steps so that its keys' fragments are worth fetching
    const int steps = (n_rows + 32 * t.rw - 1) / (32 * t.rw);
    int64_t g = units >= 1024 ? 1 : (1024 + units - 1) / units;
    if (g > (steps + 7) / 8) g = (steps + 7) / 8;
    t.pieces = (int)(g < 1 ? 1 : g);
    return t;
}

template <int D>
static void launch_weights(const WeightParams& p, int mod, int rw, dim3 grid, hipStream_t stream) {
#define LV_W(M, R) hipLaunchKernelGGL((lv_key_weights_kernel<D, M, R>), grid, dim3(256), 0, stream, p)
    switch (mod) {
        case 0: if (rw == 1) LV_W(0, 1); else LV_W(0, 2); break;
        case LV_SCORE_CAP: if (rw == 1) LV_W(LV_SCORE_CAP, 1); else LV_W(LV_SCORE_CAP, 2); break;
        case LV_SCORE_BIAS: if (rw == 1) LV_W(LV_SCORE_BIAS, 1); else LV_W(LV_SCORE_BIAS, 2); break;
        default: if (rw == 1) LV_W(3, 1); else LV_W(3, 2);
    }
#undef LV_W
}

extern "C" int64_t lv_key_weights_workspace_bytes(int batch, int n, int rows, int hq, int hkv) {
    if (batch <= 0 || n <= 0 || rows < n || hq <= 0 || hkv <= 0 || hq % hkv) return 0;
    const WeightPlan t = weight_plan(batch, n, rows, hq, hkv);
    return t.pieces > 1 ? (int64_t)t.pieces * batch * hkv * rows * (int64_t)sizeof(float) : 0;
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
    if (k_bs < 0 || (k_bs & 7) || parents_bs < 0) return lv_fail(LV_EINVAL, "lv_key_weights: batch strides must not be negative, K's a multiple of 8 elements");
    if (!(softcap >= 0.f) || softcap > 1e30f) return lv_fail(LV_EINVAL, "lv_key_weights: softcap %g must be a finite number above 0 (0: no cap)", (double)softcap);
    if (!(softmax_scale > -1e30f && softmax_scale < 1e30f)) return lv_fail(LV_EINVAL, "lv_key_weights: softmax_scale is not finite");
    const WeightPlan t = weight_plan(batch, n, rows, hq, hkv);
    const int64_t need = lv_key_weights_workspace_bytes(batch, n, rows, hq, hkv);
    if (need && !workspace) return lv_fail(LV_EINVAL, "lv_key_weights: null workspace");
    if (workspace_bytes < need) return lv_fail(LV_ESIZE, "lv_key_weights: %lld bytes of workspace needed, room for %lld", (long long)need, (long long)workspace_bytes);
    const int64_t blocks = (int64_t)batch * hkv * t.key_blocks * t.pieces;
    if (blocks > 0x7fffffffLL || (int64_t)batch * hkv > 65535) return lv_fail(LV_EINVAL, "lv_key_weights: grid too large");
    WeightParams p{};
    p.q = (const __bf16*)q; p.k = (const __bf16*)k; p.lse = lse; p.row_weight = row_weight; p.w_in = w_in; p.w_out = w_out;
    p.cache_lens = cache_lens; p.parents = parents; p.parents_bs = parents_bs; p.part = (float*)workspace;
    p.batch = batch; p.n = n; p.rows = rows; p.hq = hq; p.hkv = hkv; p.group = hq / hkv; p.pieces = t.pieces;
    p.q_bs = q_bs; p.q_ns = q_ns; p.q_hs = q_hs; p.k_bs = k_bs; p.k_rs = k_rs; p.k_hs = k_hs;
    p.wi_bs = wi_bs; p.wi_hs = wi_hs; p.wo_bs = wo_bs; p.wo_hs = wo_hs;
    p.scale_log2e = softmax_scale * 1.4426950408889634f;
    p.score = lv_score_rule(softmax_scale, softcap, slopes);
    const int mod = lv_score_mod(softcap, slopes) & (LV_SCORE_CAP | LV_SCORE_BIAS);
    if (d == 128) launch_weights<128>(p, mod, t.rw, dim3((unsigned)blocks), (hipStream_t)stream);
    else launch_weights<64>(p, mod, t.rw, dim3((unsigned)blocks), (hipStream_t)stream);
    if (hipGetLastError() != hipSuccess) return lv_fail(LV_ELAUNCH, "lv_key_weights: launch failed");
    if (t.pieces > 1)
        hipLaunchKernelGGL(lv_key_weights_join_kernel, dim3((unsigned)((rows + 255) / 256), (unsigned)(batch * hkv)), dim3(256), 0, (hipStream_t)stream, p, t.key_block);
    return hipGetLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "lv_key_weights: launch failed");
}
