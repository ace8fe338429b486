// g4_attn_tile.h -- what the attention kernels on 32 x 32 x 16 products share:
// fp32 operands as sums of terms of 16 bits, the scales of split rows and what
// weights lose by them, the order of products and LDS reads, rows to and from
// memory through LDS.
#pragma once
#include <float.h>
#include <math.h>

#include "g4_tile.h"

namespace g4 {
namespace {

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
typedef float f16_t __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ f16_t mfma32(h8_t a, h8_t b, f16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16_t mfma32(b8_t a, b8_t b, f16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// A float is the sum of three bf16: its leading 8, middle 8 and last 8 bits.
// Every product of two such terms is exact, so that matrix instructions on 16
// bits give the fp32 product.
__device__ __forceinline__ uint32_t hi_halves(uint32_t x0, uint32_t x1) { return __builtin_amdgcn_perm(x1, x0, 0x07060302u); }
__device__ __forceinline__ float rest(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
template <int NT>
__device__ __forceinline__ void split_pair(float x0, float x1, uint32_t (&t)[NT]) {
#pragma unroll
    for (int i = 0; i < NT; i++) {
        t[i] = hi_halves(__float_as_uint(x0), __float_as_uint(x1));
        if (i + 1 < NT) {
            x0 = rest(x0);
            x1 = rest(x1);
        }
    }
}
__device__ __forceinline__ b8_t as_b8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(b8_t, make_uint4(a, b, c, d));
}

// biased exponent of a row's largest magnitude -> the scale that brings it
// to [2^14, 2^15) and its inverse; low: the smallest exponent told apart
__device__ __forceinline__ float row_scale(int e) { return __uint_as_float((unsigned)(268 - e) << 23); }
__device__ __forceinline__ float row_scale_inv(int e) { return __uint_as_float((unsigned)(e - 14) << 23); }
constexpr int kLowK = 15;    // 2^-126 is a normal number
constexpr int kLowV = 51;    // sums of 2^-e stay in range

// fp32: a row's weight sum l is taken of the weights w = 2^u, u = score + e -
// maximum, that the second product needs, each times its key's 2^-e.  Where V
// rows lie far apart (zeros, with e = -90, beside 2^62) w can be below 2^-126
// and be 0 while w 2^-e is not small in l at all: the key's share of l, which
// is right whatever the exponents.  A tile holds 2^(48 - 126) times its largest
// 2^-e: from that l on what its keys can lose is below 2^-48 of l each and
// changes no bit of it, so that whether the lost shares are added, by any
// lane's need, does not show in the others.  (The comparison, a tile: fp32 of 256
// 761 -> 771 us, of 512 1607 -> 1635 over four prompts of 4096.)
__device__ __forceinline__ float lost_weight(float u, float e, float vinv) {
    if (!(u < -126.0f && u > -400.0f)) return 0.0f;
    const float k = floorf(u);   // u - k is exact
    return __builtin_ldexpf(__builtin_amdgcn_exp2f(u - k), (int)k - (int)e) - __builtin_amdgcn_exp2f(u) * vinv;
}
// l brought from maximum m to m + |d|: in two steps, as l may be as far above its
// products as 2^203
__device__ __forceinline__ float move_sum(float l, float d) {
    return l * exp2f(fmaxf(d, -100.0f)) * exp2f(fminf(d + 100.0f, 0.0f));
}

// asks for an order of a run of products and the LDS reads of their operands:
// AHEAD steps' reads before the first product, then each step's NM products
// followed by the NR reads of a later step (fp32 256: 931 -> 868 us over four
// prompts of 4096)
template <int STEPS, int AHEAD, int NM, int NR>
__device__ __forceinline__ void order_products() {
    constexpr int A = AHEAD < STEPS ? AHEAD : STEPS;
    __builtin_amdgcn_sched_group_barrier(0x100, A * NR, 0);   // LDS reads
#pragma unroll
    for (int i = 0; i < STEPS - A; i++) {
        __builtin_amdgcn_sched_group_barrier(0x8, NM, 0);     // products
        __builtin_amdgcn_sched_group_barrier(0x100, NR, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, A * NM, 0);
}

// A run of STEPS steps of products whose operands are read from LDS AHEAD steps
// before: read(i, x) reads step i's operands, use(i, x) multiplies them.  The
// scheduling barriers hold the reads where they are, where one wave a SIMD has
// registers for it (fp32 512: 2056 -> 1886 us over four prompts of 4096; the
// two-wave kernels lose 4-8 % by it).
template <typename X, int STEPS, int AHEAD, typename Read, typename Use>
__device__ __forceinline__ void run_products(Read read, Use use) {
    constexpr int N = (AHEAD < STEPS ? AHEAD : STEPS - 1) + 1;
    X x[N];
#pragma unroll
    for (int i = 0; i < N - 1; i++) read(i, x[i]);
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        if (i + N - 1 < STEPS) read(i + N - 1, x[(i + N - 1) % N]);
        __builtin_amdgcn_sched_barrier(0);
        use(i, x[i % N]);
    }
    __builtin_amdgcn_sched_barrier(0);
}

template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// between a wave's own LDS accesses, which the CU keeps in order: for the compiler
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Rows to and from memory go through LDS as whole lines: an instruction costs
// the CU's address unit four cycles for every 128-byte line it touches, and the
// operands' own order (16 bytes of each of 32 rows) touches 32 of them: 16000
// cycles for a workgroup's q and as many for its output, of the 95000 that 17
// tiles take.  (Prompts of 100 to 2048 rows with a window of 512, 8 heads of
// 256: fp32 86 -> 79 us, bf16 51 -> 44 us.)  Chunk c (16 bytes) of row r lies in
// slot c ^ r, so that neither order has bank conflicts.
template <int C>
__device__ __forceinline__ int row_slot(int r, int c) {
    return (r * C + (c ^ (r & (C < 32 ? C - 1 : 31)))) * 16;
}
struct AsTheyAre {
    __device__ __forceinline__ f4_t operator()(const f4_t& x) const { return x; }
};
// N rows of C chunks each, from `first` on, by one wave: at(r) is row r's
// address, box takes C chunks a row; edit: of 16 bytes, on the way
template <int C, int N, typename At, typename Edit = AsTheyAre>
__device__ __forceinline__ void rows_to_lds(uint8_t* box, int first, At at, int lane = threadIdx.x & 63, Edit edit = {}) {
    constexpr int K = N * C / 64;
    f4_t x[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int p = k * 64 + lane;
        x[k] = reinterpret_cast<const f4_t*>(at(first + p / C))[p % C];
    }
    wave_lds_order();
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int p = k * 64 + lane;
        *reinterpret_cast<f4_t*>(box + row_slot<C>(first + p / C, p % C)) = edit(x[k]);
    }
    wave_lds_order();
}
// the other way: 32 rows of C chunks, the first n of them
template <int C, typename At>
__device__ __forceinline__ void rows_from_lds(const uint8_t* box, int n, At at) {
    constexpr int K = C / 2, B = K < 16 ? K : 16;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));   // addresses of its own: none kept from rows_to_lds over all tiles
    wave_lds_order();
#pragma unroll
    for (int k = 0; k < K; k += B) {
        f4_t x[B];
#pragma unroll
        for (int i = 0; i < B; i++) {
            const int p = (k + i) * 64 + lane;
            x[i] = *reinterpret_cast<const f4_t*>(box + row_slot<C>(p / C, p % C));
        }
#pragma unroll
        for (int i = 0; i < B; i++) {
            const int p = (k + i) * 64 + lane;
            if (p / C < n) reinterpret_cast<f4_t*>(at(p / C))[p % C] = x[i];
        }
    }
}

}  // namespace
}  // namespace g4
