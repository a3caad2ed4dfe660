// What the kernels over a batch of ragged KV caches share: the list of key tiles of all sequences and how it is dealt to
// workgroups, the draft tree in LDS, direct global -> LDS loads.
#pragma once
#include "internal.h"

typedef __attribute__((address_space(3))) char lds_char;

template <int D>
__device__ __forceinline__ int list_lds_off(int row, int chunk) {
    if constexpr (D == 128) return lds_off128(row, chunk);
    else return lds_off64(row, chunk);
}

#define LV_TREE_UNUSED (-2)   // parents[] entry of a slot that holds no token

// cached keys of sequence s: never outside the cache, whatever the caller's array says
__device__ __forceinline__ int list_len(const int32_t* cache_lens, int s, int rows, int n) { return min(max(cache_lens[s], 0), rows - n); }

// cum[s] = tiles of sequences 0 .. s, lens[s] (one wave); returns after a barrier of the whole workgroup.  Taking up a sequence
// costs a workgroup about as much as LEAD tiles (drain, first loads, join); so that no share gets its fair part of the tiles and
// the restarts on top, every sequence but the first counts LEAD tiles more, ahead of its own: list_lead(s) of them hold no keys.
template <int LEAD>
__device__ __forceinline__ int list_lead(int s) { return s ? LEAD : 0; }
template <int BN, int LEAD>
__device__ __forceinline__ void list_scan(const int32_t* cache_lens, int batch, int rows, int n, int* cum, int* lens) {
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int carry = 0;
        for (int s0 = 0; s0 < batch; s0 += 64) {
            const int len = s0 + lane < batch ? list_len(cache_lens, s0 + lane, rows, n) : 0;
            int x = s0 + lane < batch ? (len + n + BN - 1) / BN + list_lead<LEAD>(s0 + lane) : 0;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int y = __shfl_up(x, off);
                if (lane >= off) x += y;
            }
            if (s0 + lane < batch) {
                cum[s0 + lane] = carry + x;
                if (lens) lens[s0 + lane] = len;
            }
            carry += __shfl(x, 63);
        }
    }
    __syncthreads();
}

// The list dealt to the shares: `total` tiles, the first total % G shares one more than the rest.
struct ListDeal {
    uint32_t G, each, extra;
    __device__ ListDeal(uint32_t shares, uint32_t total) : G(min(shares, total)), each(total / G), extra(total - each * G) {}
    __device__ int first(uint32_t g) const { return (int)(g * each + min(g, extra)); }
    __device__ int share_of(uint32_t tile) const {
        const uint32_t head = extra * (each + 1);
        return (int)(tile < head ? tile / (each + 1) : extra + (tile - head) / each);
    }
};

// Direct global -> LDS load, 16 bytes per lane, lane i -> LDS byte lds_dst + 16 i (M0 carries lds_dst; nothing else in the kernels
// that use it needs M0, so it is not restored).  As asm so that the compiler does not count it; completion is waited for by
// hand.
__device__ __forceinline__ void list_dma16(__amdgpu_buffer_rsrc_t rs, int voff, uint32_t lds_dst) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rs), "s"(lds_dst) : "memory");
}

// parents[] of a sequence -> par (checked), depth of every token and, when asked for, its ancestors' bits [n][words] (itself
// among them).  The whole workgroup (nt threads); barriers before, between and after.
__device__ __forceinline__ void list_tree(const int32_t* parents, int n, int words, bool bits, int* par, int* depth, uint32_t* anc, int tid, int nt) {
    __syncthreads();                  // the previous sequence's arrays are no longer read
    for (int i = tid; i < n; i += nt) {
        const int x = parents[i];
        par[i] = x < i ? x : -1;      // a parent stands before its child: the walk below always ends
    }
    __syncthreads();
    for (int i = tid; i < n; i += nt) {
        if (bits)
            for (int x = 0; x < words; ++x) anc[i * words + x] = 0;
        int dep = -1, at = i;
        if (par[i] != LV_TREE_UNUSED)
            while (at >= 0) {
                if (bits) anc[i * words + (at >> 5)] |= 1u << (at & 31);
                ++dep;
                at = par[at];
                if (at >= 0 && par[at] == LV_TREE_UNUSED) at = -1;      // a parent that holds no token is none
            }
        depth[i] = max(dep, 0);
    }
    __syncthreads();
}
