// g4_kvpage.h -- the paged KV cache's layout, shared by the kernels that
// write it, read it back and attend over it.
//
// A pool holds n_pages pages of `page` tokens (a power of two from 16 up);
// K and V are pools of their own.  Page p, kv head h, 16-token block b:
// 16 * hd elements at ((p * n_kv + h) * (page / 16) + b) * 16 * hd.  A block is
// stored in the order in which the matrix cores take it, in pieces of 64 lanes
// x 16 bytes, so that a wave reads a block as whole contiguous kilobytes and
// has its operands in registers without a move:
//   K (operand rows = tokens): lane 16 g + t of piece c holds token t's dims
//     (4 c + g) * E .. + E - 1, E = 16 / element size;
//   V (operand rows = dims): lane 16 g + n of piece c holds, for each
//     i < 4 / element size (1 for F32, 2 for 16 bits, 4 for codes), dim
//     (64 / element size) c + 16 i + n of tokens 4 g .. 4 g + 3: the lane
//     group that gets the scores of tokens 4 g .. 4 g + 3 out of the first
//     product holds their V.
// Q8: behind the codes, one fp32 scale for each page, kv head and token.
#pragma once
#include "g4_device.h"
#include "g4_internal.h"

namespace g4 {

constexpr int kKvMaxPage = 4096;
constexpr int kKvMaxSeqs = 4096;

inline int kv_elem_size(int type) {
    return type == G4_F32 ? 4 : type == G4_F16 || type == G4_BF16 ? 2 : type == G4_KV_Q8 ? 1 : 0;
}

// byte of (token t of 16, dim d) in a K / V block of elements of ES bytes
template <int ES>
__device__ __forceinline__ int kv_k_byte(int t, int d) {
    constexpr int E = 16 / ES;
    return (d / (4 * E) * 64 + (d / E) % 4 * 16 + t) * 16 + d % E * ES;
}
template <int ES>
__device__ __forceinline__ int kv_v_byte(int t, int d) {
    constexpr int D = 64 / ES;   // dims of a piece
    return (d / D * 64 + t / 4 * 16 + d % 16) * 16 + (d % D / 16 * 4 + t % 4) * ES;
}

// where the pages of the sequences are
struct KvPool {
    uint8_t* kp;
    uint8_t* vp;
    const int* table;
    int table_stride, n_pages, lgpage, n_kv;
    size_t scale_off;   // Q8: bytes before the scales
    // page that holds position pos of sequence s (which the caller has
    // checked against table_stride), -1 if the table's entry is not a page
    __device__ __forceinline__ int page_of(int s, int pos) const {
        const int p = table[(size_t)s * table_stride + (pos >> lgpage)];
        return p >= 0 && p < n_pages ? p : -1;
    }
    // 16-token block of position pos in page p, counted over the pool
    __device__ __forceinline__ size_t block_of(int p, int h, int pos) const {
        return (((size_t)p * n_kv + h) << (lgpage - 4)) + ((pos & ((1 << lgpage) - 1)) >> 4);
    }
    // positions 0 .. len - 1 have entries in the table
    __device__ __forceinline__ bool fits(int len) const {
        return len >= 0 && (len == 0 || (len - 1) >> lgpage < table_stride);
    }
};

// the sequence that work unit u belongs to: the largest s < n with
// (mul cu[s] >> lg) + extra * s <= u (0 if there is none), found by a whole
// wave in steps of 64 candidates.  Any contents of cu give an s in range.
__device__ __forceinline__ unsigned unit_base(const int* __restrict__ cu, int s, int mul, int lg, int extra) {
    return (unsigned)(((unsigned long long)(unsigned)cu[s] * (unsigned)mul) >> lg) + (unsigned)extra * (unsigned)s;
}
__device__ __forceinline__ int unit_seq(const int* __restrict__ cu, int n, int mul, int lg, int extra, unsigned u) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    while (n > 1) {
        const int step = (n + 63) >> 6;
        bool in = (long)lane * step < n;
        if (in) in = unit_base(cu, lo + lane * step, mul, lg, extra) <= u;
        const int c = __popcll(__ballot(in));
        const int adv = (c > 0 ? c - 1 : 0) * step;
        lo += adv;
        n = n - adv < step ? n - adv : step;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// that sequence with its rows and (lens given) its length.  Up to 64 sequences
// all of it is in the lanes after one round trip to memory.
struct SeqAt {
    int s, r0, r1, len;
};
__device__ __forceinline__ SeqAt find_seq(const int* __restrict__ cu, const int* __restrict__ lens, int n, int mul, int lg,
                                          int extra, unsigned u) {
    SeqAt r;
    if (n <= 64) {
        const int lane = threadIdx.x & 63, i = lane < n ? lane : n - 1;
        const int c0 = cu[i], c1 = cu[i + 1], len = lens ? lens[i] : 0;
        const unsigned base = (unsigned)(((unsigned long long)(unsigned)c0 * (unsigned)mul) >> lg) + (unsigned)extra * (unsigned)i;
        const int c = __popcll(__ballot(lane < n && base <= u));
        r.s = c > 0 ? c - 1 : 0;
        r.r0 = __builtin_amdgcn_readlane(c0, r.s);
        r.r1 = __builtin_amdgcn_readlane(c1, r.s);
        r.len = __builtin_amdgcn_readlane(len, r.s);
    } else {
        r.s = unit_seq(cu, n, mul, lg, extra, u);
        r.r0 = cu[r.s];
        r.r1 = cu[r.s + 1];
        r.len = lens ? lens[r.s] : 0;
    }
    return r;
}

// host: whether a launch may have that many workgroups
inline bool kv_grid_fits(size_t wgs, int threads) { return wgs < ((size_t)1 << 32) / threads; }

// host: the arguments every entry point of the cache checks alike
int kv_pool_check(const char* who, KvPool* o, const void* kp, const void* vp, int type, int n_pages, int page, int n_kv,
                  int hd, const int* table, int table_stride);

}  // namespace g4
