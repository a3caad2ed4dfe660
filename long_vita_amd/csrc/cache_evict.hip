// A KV cache cut down to its first, last and heaviest keys, for gfx950.
//
//   per sequence and KV head, len > keep: rows [0, sink), rows [len - recent, len), and of the rows between the
//   keep - sink - recent with the largest weight (ties: the lower row), all in their old order; len <= keep: every row
//
// The choice is a radix select: weights become unsigned keys that order as the numbers do (NaN above everything, as a sort
// puts it; -0 equal to 0), the threshold is found digit by digit from histograms, and what lies above it, plus the first few
// equal to it, is numbered by counting.  Counts are integers, so the order in which they are added does not matter.  Caches of
// up to 16,384 rows: one workgroup per head holds all keys in registers and does everything in LDS, one launch.  Longer ones:
// workgroups of 2,048 rows, six short launches, each a read of the weights (which stay in the last-level cache).
// Then the kept rows are gathered; that is where the bytes are: K and V, read and written once.
//
// Measured, 8 heads of 128: 262,144 rows to 65,536 in 132 us (gather 86 us, 4.6 TB/s); 8 caches of up to 4,096 rows to 1,024 in
// 23 us (11 us to choose, 12 us to gather).
#include "internal.h"
#include "../../include/lvattn.h"

#define LV_EVICT_SMALL 16384
#define LV_EVICT_CHUNK 2048

__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.f);          // -0 -> 0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct EvictRange { int len, lo, hi, want; bool cut; };   // rows [lo, hi) compete for `want` places
__device__ __forceinline__ EvictRange evict_range(const EvictParams& p, int s) {
    EvictRange e;
    e.len = min(max(p.cache_lens[s], 0), p.rows);
    e.cut = e.len > p.keep;
    e.lo = p.sink;
    e.hi = e.len - p.recent;
    e.want = p.keep - p.sink - p.recent;
    return e;
}

// ---------------------------------------------------------------------------
// up to 1024 PER rows: 1024 threads, row 1024 i + tid in register i
// ---------------------------------------------------------------------------
template <int PER>
__global__ __launch_bounds__(1024) void lv_evict_small_kernel(EvictParams p) {
    constexpr int COPIES = 8;                       // of the histogram: lanes that hit one bin are spread over them
    __shared__ uint32_t hist[COPIES][257];
    __shared__ uint32_t digit_s, left_s;
    __shared__ uint32_t cnt[PER * 16];              // per (register, wave)
    __shared__ uint32_t wsum[16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int s = blockIdx.x / p.hkv, kvh = blockIdx.x % p.hkv;
    const EvictRange e = evict_range(p, s);
    int32_t* idx = p.index + (int64_t)blockIdx.x * p.keep;
    if (kvh == 0 && tid == 0 && p.new_lens) p.new_lens[s] = min(e.len, p.keep);
    if (!e.cut) {
        for (int i = tid; i < p.keep; i += 1024) idx[i] = i < e.len ? i : -1;
        return;
    }
    const float* wt = p.w_in + (int64_t)s * p.wi_bs + (int64_t)kvh * p.wi_hs;
    uint32_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = 1024 * i + tid;
        key[i] = (j >= e.lo && j < e.hi) ? order_key(wt[j]) : 0u;
    }
    // threshold: the want-th largest key, digit by digit
    uint32_t prefix = 0, left = (uint32_t)e.want;   // keys above the prefix still to be found
    if (e.want > 0) {
#pragma unroll 1
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < COPIES * 257; i += 1024) (&hist[0][0])[i] = 0;
            __syncthreads();
            const uint32_t himask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int j = 1024 * i + tid;
                if (j >= e.lo && j < e.hi && (key[i] & himask) == prefix) atomicAdd(&hist[lane & (COPIES - 1)][(key[i] >> shift) & 255], 1u);
            }
            __syncthreads();
            if (w == 0) {                           // from the top digit down: the one where the count reaches `left`
                uint32_t c[4], mine = 0;
#pragma unroll
                for (int x = 0; x < 4; ++x) {       // lane l: digits 255 - 4l - x
                    c[x] = 0;
#pragma unroll
                    for (int y = 0; y < COPIES; ++y) c[x] += hist[y][255 - 4 * lane - x];
                    mine += c[x];
                }
                uint32_t incl = mine;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const uint32_t y = __shfl_up(incl, off);
                    if (lane >= off) incl += y;
                }
                uint32_t before = incl - mine;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (before < left && before + c[x] >= left) {
                        digit_s = 255 - 4 * lane - x;
                        left_s = left - before;
                    }
                    before += c[x];
                }
            }
            __syncthreads();
            prefix |= digit_s << shift;
            left = left_s;
            __syncthreads();
        }
    }
    // rows equal to the threshold: the first `left` of them stay.  Count them per (register, wave), scan, then the same for
    // the rows that stay
    uint32_t base[PER];
#pragma unroll 1
    for (int round = 0; round < 2; ++round) {
        bool f[PER];
        uint32_t below[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int j = 1024 * i + tid;
            const bool mid = j >= e.lo && j < e.hi;
            if (round == 0) f[i] = mid && e.want > 0 && key[i] == prefix;
            else {
                const bool eq = mid && e.want > 0 && key[i] == prefix;
                f[i] = j < e.len && (!mid || (e.want > 0 && (key[i] > prefix || (eq && base[i] < left))));
            }
            const uint64_t m = __ballot(f[i]);
            below[i] = __popcll(m & ((1ull << lane) - 1));
            if (lane == 0) cnt[i * 16 + w] = __popcll(m);
        }
        __syncthreads();
        if (tid < PER * 16) {                       // exclusive scan of the counts, a wave to 64 of them
            const uint32_t mine = cnt[tid];
            uint32_t incl = mine;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t y = __shfl_up(incl, off);
                if (lane >= off) incl += y;
            }
            if (lane == 63) wsum[w] = incl;
            cnt[tid] = incl - mine;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = i * 16 + w;
            uint32_t off = cnt[at] + below[i];
#pragma unroll
            for (int x = 0; x < PER * 16 / 64; ++x)
                if (x < at / 64) off += wsum[x];
            base[i] = off;
            if (round == 1 && f[i]) idx[off] = 1024 * i + tid;     // exactly `keep` rows stay: off < keep
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// longer caches: histograms of 11, 11 and 10 bits over all chunks, then counts per chunk, then the numbering
// ---------------------------------------------------------------------------
struct Select { uint32_t prefix, left; };
__device__ __forceinline__ int digit_shift(int pass) { return pass == 0 ? 21 : (pass == 1 ? 10 : 0); }
__device__ __forceinline__ int digit_bits(int pass) { return pass == 2 ? 10 : 11; }

// digits 0 .. passes-1 of the threshold, from the finished histograms (256 threads; every workgroup for itself)
__device__ __forceinline__ Select evict_select(const EvictParams& p, int bh, int want, int passes) {
    __shared__ uint32_t pick[2], part[4];
    Select sel = {0u, (uint32_t)want};
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    for (int pass = 0; pass < passes; ++pass) {
        const uint32_t* hist = p.hist + ((int64_t)pass * p.batch * p.hkv + bh) * 2048;
        const int per = (1 << digit_bits(pass)) / 256;             // digits per thread: 8 or 4, from the top down
        uint32_t c[8], mine = 0;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            c[x] = x < per ? hist[(1 << digit_bits(pass)) - 1 - per * tid - x] : 0u;
            mine += c[x];
        }
        uint32_t incl = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t y = __shfl_up(incl, off);
            if (lane >= off) incl += y;
        }
        if (lane == 63) part[w] = incl;
        __syncthreads();
        uint32_t before = incl - mine;
        for (int x = 0; x < w; ++x) before += part[x];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            if (x < per && before < sel.left && before + c[x] >= sel.left) {
                pick[0] = (1 << digit_bits(pass)) - 1 - per * tid - x;
                pick[1] = sel.left - before;
            }
            before += c[x];
        }
        __syncthreads();
        sel.prefix |= pick[0] << digit_shift(pass);
        sel.left = pick[1];
        __syncthreads();
    }
    return sel;
}

__global__ __launch_bounds__(256) void lv_evict_clear_kernel(EvictParams p) {
    const int64_t n = (int64_t)3 * p.batch * p.hkv * 2048;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p.hist[i] = 0;
}

__global__ __launch_bounds__(256) void lv_evict_hist_kernel(EvictParams p, int pass) {
    constexpr int COPIES = 2;
    constexpr int PER = LV_EVICT_CHUNK / 256;
    __shared__ uint32_t hist[COPIES][2049];
    const int bh = blockIdx.y, s = bh / p.hkv, kvh = bh % p.hkv, tid = threadIdx.x;
    const EvictRange e = evict_range(p, s);
    const int c0 = blockIdx.x * LV_EVICT_CHUNK, c1 = min(c0 + LV_EVICT_CHUNK, e.hi);
    if (!e.cut || e.want <= 0 || c0 >= e.hi) return;
    const float* wt = p.w_in + (int64_t)s * p.wi_bs + (int64_t)kvh * p.wi_hs;
    float x[PER];                                                  // on their way while the threshold's digits so far are found
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = c0 + 256 * i + tid;
        x[i] = j >= e.lo && j < c1 ? wt[j] : 0.f;
    }
    for (int i = tid; i < COPIES * 2049; i += 256) (&hist[0][0])[i] = 0;
    const Select sel = evict_select(p, bh, e.want, pass);
    __syncthreads();
    const uint32_t himask = pass == 0 ? 0u : 0xffffffffu << (digit_shift(pass) + digit_bits(pass));
    const uint32_t dmask = (1u << digit_bits(pass)) - 1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = c0 + 256 * i + tid;
        const uint32_t key = order_key(x[i]);
        if (j >= e.lo && j < c1 && (key & himask) == sel.prefix) atomicAdd(&hist[tid & (COPIES - 1)][(key >> digit_shift(pass)) & dmask], 1u);
    }
    __syncthreads();
    uint32_t* out = p.hist + ((int64_t)pass * p.batch * p.hkv + bh) * 2048;
    for (int i = tid; i < (1 << digit_bits(pass)); i += 256) {
        uint32_t x = 0;
#pragma unroll
        for (int y = 0; y < COPIES; ++y) x += hist[y][i];
        if (x) atomicAdd(out + i, x);                               // whole numbers: any order gives the same sum
    }
}

// 0: rows above the threshold or outside the competition, 1: rows equal to it
__device__ __forceinline__ int evict_class(const EvictRange& e, const Select& sel, int j, float wgt) {
    if (j >= e.len) return -1;
    if (j < e.lo || j >= e.hi) return 0;
    if (e.want <= 0) return -1;
    const uint32_t key = order_key(wgt);
    return key > sel.prefix ? 0 : (key == sel.prefix ? 1 : -1);
}

// rows of a chunk in each class -> counts [bh][chunks][2]; the threshold -> thr [bh][2]
__global__ __launch_bounds__(256) void lv_evict_count_kernel(EvictParams p) {
    const int bh = blockIdx.y, s = bh / p.hkv, kvh = bh % p.hkv, tid = threadIdx.x;
    const EvictRange e = evict_range(p, s);
    if (!e.cut) return;
    constexpr int PER = LV_EVICT_CHUNK / 256;
    const float* wt = p.w_in + (int64_t)s * p.wi_bs + (int64_t)kvh * p.wi_hs;
    float x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = blockIdx.x * LV_EVICT_CHUNK + 256 * i + tid;
        x[i] = j < e.len ? wt[j] : 0.f;
    }
    const Select sel = evict_select(p, bh, e.want, e.want > 0 ? 3 : 0);
    uint32_t n0 = 0, n1 = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int c = evict_class(e, sel, blockIdx.x * LV_EVICT_CHUNK + 256 * i + tid, x[i]);
        n0 += __popcll(__ballot(c == 0));
        n1 += __popcll(__ballot(c == 1));
    }
    __shared__ uint32_t t0[4], t1[4];
    if ((tid & 63) == 0) { t0[tid >> 6] = n0; t1[tid >> 6] = n1; }
    __syncthreads();
    if (tid == 0) {
        uint32_t* out = p.counts + ((int64_t)bh * p.chunks + blockIdx.x) * 2;
        out[0] = t0[0] + t0[1] + t0[2] + t0[3];
        out[1] = t1[0] + t1[1] + t1[2] + t1[3];
        if (blockIdx.x == 0) { p.thr[2 * bh] = sel.prefix; p.thr[2 * bh + 1] = sel.left; }
    }
}

// the kept rows' numbers: a thread owns 8 consecutive rows of the chunk
__global__ __launch_bounds__(256) void lv_evict_index_kernel(EvictParams p) {
    constexpr int PER = LV_EVICT_CHUNK / 256;
    __shared__ float tile[LV_EVICT_CHUNK + LV_EVICT_CHUNK / 32];      // (one word in 33 unused: a thread's rows are 8 apart)
    __shared__ uint32_t sum0[4], sum1[4];
    const int bh = blockIdx.y, s = bh / p.hkv, kvh = bh % p.hkv, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const EvictRange e = evict_range(p, s);
    int32_t* idx = p.index + (int64_t)bh * p.keep;
    const int c0 = blockIdx.x * LV_EVICT_CHUNK;
    if (blockIdx.x == 0 && kvh == 0 && tid == 0 && p.new_lens) p.new_lens[s] = min(e.len, p.keep);
    if (!e.cut) {
        for (int i = c0 + tid; i < min(c0 + LV_EVICT_CHUNK, p.keep); i += 256) idx[i] = i < e.len ? i : -1;
        // (keep <= rows: the chunks of the rows cover the index)
        return;
    }
    if (c0 >= e.len) return;
    const Select sel = {p.thr[2 * bh], p.thr[2 * bh + 1]};
    const float* wt = p.w_in + (int64_t)s * p.wi_bs + (int64_t)kvh * p.wi_hs;
#pragma unroll 8
    for (int i = 0; i < PER; ++i) {
        const int x = 256 * i + tid;
        tile[x + x / 32] = c0 + x < e.len ? wt[c0 + x] : 0.f;
    }
    // rows of both classes in the chunks before this one
    uint32_t b0 = 0, b1 = 0;
    for (int c = tid; c < (int)blockIdx.x; c += 256) {
        b0 += p.counts[((int64_t)bh * p.chunks + c) * 2];
        b1 += p.counts[((int64_t)bh * p.chunks + c) * 2 + 1];
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { b0 += __shfl_xor(b0, off); b1 += __shfl_xor(b1, off); }
    if (lane == 0) { sum0[w] = b0; sum1[w] = b1; }
    __syncthreads();
    b0 = sum0[0] + sum0[1] + sum0[2] + sum0[3];
    b1 = sum1[0] + sum1[1] + sum1[2] + sum1[3];
    __syncthreads();
    uint32_t mask0 = 0, mask1 = 0;
#pragma unroll 8
    for (int i = 0; i < PER; ++i) {
        const int x = PER * tid + i;
        const int c = evict_class(e, sel, c0 + x, tile[x + x / 32]);
        mask0 |= (c == 0 ? 1u : 0u) << i;
        mask1 |= (c == 1 ? 1u : 0u) << i;
    }
    uint32_t i0 = __popc(mask0), i1 = __popc(mask1);
    const uint32_t m0 = i0, m1 = i1;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t y0 = __shfl_up(i0, off), y1 = __shfl_up(i1, off);
        if (lane >= off) { i0 += y0; i1 += y1; }
    }
    if (lane == 63) { sum0[w] = i0; sum1[w] = i1; }
    __syncthreads();
    uint32_t at0 = b0 + i0 - m0, at1 = b1 + i1 - m1;               // rows of each class before this thread's
    for (int x = 0; x < w; ++x) { at0 += sum0[x]; at1 += sum1[x]; }
    for (int i = 0; i < PER; ++i) {
        const bool eq = (mask1 >> i) & 1, stay = ((mask0 >> i) & 1) || (eq && at1 < sel.left);
        if (stay) idx[at0 + min(at1, sel.left)] = c0 + PER * tid + i;
        at0 += (mask0 >> i) & 1;
        at1 += eq;
    }
}

// ---------------------------------------------------------------------------
// the kept rows of K, V and the weights.  16 bytes per thread; the heads of a row are neighbours, so the writes are whole rows
// of the new cache and the reads whole head rows (128 or 256 bytes) of the old one.  Every byte is touched once: the accesses ask
// for no place in the caches, and one (row, head) per group of threads leaves the most waves to wait side by side (262,144 rows
// to 65,536, 8 heads, the whole eviction: 156 us with plain accesses and four pairs per group, 142 without a place, 135 and 132
// with two and one pair).
// ---------------------------------------------------------------------------
template <int CPR>
__global__ __launch_bounds__(256) void lv_evict_take_kernel(EvictParams p) {
    const int64_t x = (int64_t)blockIdx.x * (256 / CPR) + threadIdx.x / CPR;       // row * heads + head
    if (x >= (int64_t)p.keep * p.hkv) return;
    const int s = blockIdx.y, ch = threadIdx.x % CPR, head = (int)(x % p.hkv);
    const int64_t j = x / p.hkv;
    const int src = p.index[((int64_t)s * p.hkv + head) * p.keep + j];
    if (src < 0 && !p.zero_fill) return;
    u32x4 kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
    float wx = 0.f;
    if (src >= 0) {
        kx = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.k_in + (int64_t)s * p.ki_bs + (int64_t)src * p.ki_rs + (int64_t)head * p.ki_hs + ch * 8));
        vx = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.v_in + (int64_t)s * p.vi_bs + (int64_t)src * p.vi_rs + (int64_t)head * p.vi_hs + ch * 8));
        if (ch == 0) wx = p.w_in[(int64_t)s * p.wi_bs + (int64_t)head * p.wi_hs + src];
    }
    __builtin_nontemporal_store(kx, reinterpret_cast<u32x4*>(p.k_out + (int64_t)s * p.ko_bs + j * p.ko_rs + (int64_t)head * p.ko_hs + ch * 8));
    __builtin_nontemporal_store(vx, reinterpret_cast<u32x4*>(p.v_out + (int64_t)s * p.vo_bs + j * p.vo_rs + (int64_t)head * p.vo_hs + ch * 8));
    if (ch == 0) p.w_out[(int64_t)s * p.wo_bs + (int64_t)head * p.wo_hs + j] = wx;
}

static int evict_chunks(int rows) { return (rows + LV_EVICT_CHUNK - 1) / LV_EVICT_CHUNK; }

extern "C" int64_t lv_evict_workspace_bytes(int batch, int rows, int hkv) {
    if (batch <= 0 || rows <= 0 || hkv <= 0 || rows <= LV_EVICT_SMALL) return 0;
    return (int64_t)batch * hkv * (3 * 2048 + 2 * evict_chunks(rows) + 2) * (int64_t)sizeof(uint32_t);
}

extern "C" int lv_evict_index(const float* weight, const int32_t* cache_lens, int32_t* index, int32_t* new_lens, void* workspace, int64_t workspace_bytes,
                              int batch, int rows, int hkv, int keep, int sink, int recent, int64_t w_bs, int64_t w_hs, void* stream) {
    if (!weight || !cache_lens || !index) return lv_fail(LV_EINVAL, "lv_evict_index: null weight / cache_lens / index pointer");
    if (batch <= 0 || rows <= 0 || hkv <= 0 || (int64_t)batch * hkv > 65535) return lv_fail(LV_EINVAL, "lv_evict_index: batch %d, %d rows, %d KV heads", batch, rows, hkv);
    if (keep <= 0 || keep > rows || sink < 0 || recent < 0 || (int64_t)sink + recent > keep)
        return lv_fail(LV_EINVAL, "lv_evict_index: keep %d (1 to %d rows) must hold sink %d + recent %d", keep, rows, sink, recent);
    const int64_t need = lv_evict_workspace_bytes(batch, rows, hkv);
    if (need && (!workspace || workspace_bytes < need))
        return lv_fail(LV_ESIZE, "lv_evict_index: %lld bytes of workspace needed, room for %lld", (long long)need, (long long)(workspace ? workspace_bytes : 0));
    EvictParams p{};
    p.w_in = weight; p.cache_lens = cache_lens; p.index = index; p.new_lens = new_lens;
    p.batch = batch; p.rows = rows; p.hkv = hkv; p.keep = keep; p.sink = sink; p.recent = recent; p.wi_bs = w_bs; p.wi_hs = w_hs;
    hipStream_t st = (hipStream_t)stream;
    if (rows <= LV_EVICT_SMALL) {
        if (rows <= 4096) hipLaunchKernelGGL(lv_evict_small_kernel<4>, dim3((unsigned)(batch * hkv)), dim3(1024), 0, st, p);
        else hipLaunchKernelGGL(lv_evict_small_kernel<LV_EVICT_SMALL / 1024>, dim3((unsigned)(batch * hkv)), dim3(1024), 0, st, p);
    } else {
        p.chunks = evict_chunks(rows);
        p.hist = (uint32_t*)workspace;
        p.counts = p.hist + (int64_t)3 * batch * hkv * 2048;
        p.thr = p.counts + (int64_t)batch * hkv * p.chunks * 2;
        const dim3 grid((unsigned)p.chunks, (unsigned)(batch * hkv));
        hipLaunchKernelGGL(lv_evict_clear_kernel, dim3((unsigned)(batch * hkv > 40 ? 1024 : batch * hkv * 24)), dim3(256), 0, st, p);
        for (int pass = 0; pass < 3; ++pass) hipLaunchKernelGGL(lv_evict_hist_kernel, grid, dim3(256), 0, st, p, pass);
        hipLaunchKernelGGL(lv_evict_count_kernel, grid, dim3(256), 0, st, p);
        hipLaunchKernelGGL(lv_evict_index_kernel, grid, dim3(256), 0, st, p);
    }
    return hipGetLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "lv_evict_index: launch failed");
}

extern "C" int lv_evict_take(const void* k_in, const void* v_in, const float* w_in, const int32_t* index, void* k_out, void* v_out, float* w_out, int batch,
                             int hkv, int d, int keep, int zero_fill, int64_t ki_bs, int64_t ki_rs, int64_t ki_hs, int64_t vi_bs, int64_t vi_rs,
                             int64_t vi_hs, int64_t wi_bs, int64_t wi_hs, int64_t ko_bs, int64_t ko_rs, int64_t ko_hs, int64_t vo_bs, int64_t vo_rs,
                             int64_t vo_hs, int64_t wo_bs, int64_t wo_hs, void* stream) {
    if (!k_in || !v_in || !w_in || !index || !k_out || !v_out || !w_out) return lv_fail(LV_EINVAL, "lv_evict_take: null pointer");
    if (d != 64 && d != 128) return lv_fail(LV_EINVAL, "lv_evict_take: head dim %d (64 or 128)", d);
    if (batch <= 0 || batch > 65535 || hkv <= 0 || keep <= 0) return lv_fail(LV_EINVAL, "lv_evict_take: bad sizes");
    if (((uintptr_t)k_in | (uintptr_t)v_in | (uintptr_t)k_out | (uintptr_t)v_out) & 15) return lv_fail(LV_EINVAL, "lv_evict_take: caches must be 16-byte aligned");
    if ((ki_bs | ki_rs | ki_hs | vi_bs | vi_rs | vi_hs | ko_bs | ko_rs | ko_hs | vo_bs | vo_rs | vo_hs) & 7)
        return lv_fail(LV_EINVAL, "lv_evict_take: strides must be multiples of 8 elements");
    EvictParams p{};
    p.k_in = (const __bf16*)k_in; p.v_in = (const __bf16*)v_in; p.w_in = w_in; p.index = const_cast<int32_t*>(index);
    p.k_out = (__bf16*)k_out; p.v_out = (__bf16*)v_out; p.w_out = w_out;
    p.batch = batch; p.hkv = hkv; p.keep = keep; p.zero_fill = zero_fill;
    p.ki_bs = ki_bs; p.ki_rs = ki_rs; p.ki_hs = ki_hs; p.vi_bs = vi_bs; p.vi_rs = vi_rs; p.vi_hs = vi_hs; p.wi_bs = wi_bs; p.wi_hs = wi_hs;
    p.ko_bs = ko_bs; p.ko_rs = ko_rs; p.ko_hs = ko_hs; p.vo_bs = vo_bs; p.vo_rs = vo_rs; p.vo_hs = vo_hs; p.wo_bs = wo_bs; p.wo_hs = wo_hs;
    const int per_block = 256 / (d / 8);
    const int64_t blocks = ((int64_t)keep * hkv + per_block - 1) / per_block;
    if (blocks > 0x7fffffffLL) return lv_fail(LV_EINVAL, "lv_evict_take: grid too large");
    if (d == 128) hipLaunchKernelGGL((lv_evict_take_kernel<16>), dim3((unsigned)blocks, (unsigned)batch), dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL((lv_evict_take_kernel<8>), dim3((unsigned)blocks, (unsigned)batch), dim3(256), 0, (hipStream_t)stream, p);
    return hipGetLastError() == hipSuccess ? LV_OK : lv_fail(LV_ELAUNCH, "lv_evict_take: launch failed");
}
