// g4_kvrows.h -- packed rows of sequences in blocks of the paged cache's 16
// tokens: which rows a workgroup has, how they lie in its registers, and how
// they are rounded and written into a page.
#pragma once
#include "g4_kvpage.h"

namespace g4 {
namespace {

// A workgroup's share: up to 16 rows of one sequence that fall into one
// 16-token block of the cache, of one head.
// Sequence s takes the units (cu[s] >> 4) + 2 s onwards: its n rows touch at
// most (n + 30) / 16 blocks, so the shares never overlap and no prefix sum is
// needed; units past a sequence's last block have nothing to do.
struct Unit {
    int s, at;         // sequence, position of the block's token 0
    int t0, t1;        // tokens of the block that take part
    int row;           // row of token 0 of the block (may lie before the first row)
};

// unit id of a launch.  fits(len): whether that many positions have a place
template <typename Fits>
__device__ __forceinline__ bool find_unit(const int* __restrict__ cu, const int* __restrict__ lens, int n_seqs, int m, unsigned id,
                                          Fits fits, Unit& u) {
    const SeqAt q = find_seq(cu, lens, n_seqs, 1, 4, 2, id);
    if (q.r0 < 0 || q.r1 <= q.r0 || q.r1 > m || q.r1 - q.r0 > q.len || !fits(q.len)) return false;
    const int pos0 = q.len - (q.r1 - q.r0);
    const unsigned b = id - (((unsigned)q.r0 >> 4) + 2u * (unsigned)q.s);
    const int first = pos0 >> 4, blocks = ((q.len - 1) >> 4) - first + 1;
    if (b >= (unsigned)blocks) return false;
    u.s = q.s;
    u.at = (first + (int)b) << 4;
    u.t0 = pos0 > u.at ? pos0 - u.at : 0;
    u.t1 = q.len - u.at < 16 ? q.len - u.at : 16;
    u.row = q.r0 + (u.at - pos0);
    return true;
}

template <int TYPE>
struct Elem;
template <>
struct Elem<G4_F32> {
    typedef float t;
    static __device__ __forceinline__ t of(float x) { return x; }
    static __device__ __forceinline__ float back(t x) { return x; }
};
template <>
struct Elem<G4_F16> {
    typedef _Float16 t;
    static __device__ __forceinline__ t of(float x) { return (_Float16)x; }
    static __device__ __forceinline__ float back(t x) { return (float)x; }
};
template <>
struct Elem<G4_BF16> {
    typedef __bf16 t;
    static __device__ __forceinline__ t of(float x) { return (__bf16)x; }
    static __device__ __forceinline__ float back(t x) { return (float)x; }
};
template <>
struct Elem<G4_KV_Q8> {
    typedef int8_t t;
    static __device__ __forceinline__ t of(float x) { return (int8_t)x; }
    static __device__ __forceinline__ float back(t x) { return (float)x; }
};

// rows of a block over the workgroup's four waves: LPR lanes a row, VPL float4
// a lane, RPW rows a wave and pass
template <int HD>
struct RowMap {
    static constexpr int LPR = HD / 4 < 64 ? HD / 4 : 64, VPL = HD / 4 / LPR, RPW = 64 / LPR, PASS = 4 / RPW;
};
// whether any of pass i's rows of this wave takes part
template <int HD>
__device__ __forceinline__ bool pass_in_use(const Unit& u, int i, int wave) {
    constexpr int RPW = RowMap<HD>::RPW;
    const int t = (i * 4 + __builtin_amdgcn_readfirstlane(wave)) * RPW;
    return t + RPW > u.t0 && t < u.t1;
}

// Rows of 16 tokens are rounded in registers, put into the block's order in
// LDS and written as whole 16-byte pieces; where only some of a piece's tokens
// take part (K pieces belong to one token, V pieces to four) only those are
// written.
// Q8: d = max|x| / 127 and codes rint(x / d), both fp32 divisions, so that a
// code is the nearest one and what is read back is the same wherever it is
// computed; a row with an infinity or NaN gets the scale NaN.
// x: the workgroup's rows as RowMap has them, img: 16 * HD elements of LDS.
template <int TYPE, int HD>
__device__ __forceinline__ void store_block(const KvPool& p, int page, int head, const Unit& u, bool is_v,
                                            const float4 (&x)[RowMap<HD>::PASS][RowMap<HD>::VPL], uint8_t* img) {
    typedef typename Elem<TYPE>::t T;
    constexpr int ES = sizeof(T);
    typedef RowMap<HD> M;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int sub = lane / M::LPR, col = lane % M::LPR;
    uint8_t* pool = is_v ? p.vp : p.kp;
    const size_t block = p.block_of(page, head, u.at);
#pragma unroll
    for (int i = 0; i < M::PASS; i++) {
        const int t = (i * 4 + wave) * M::RPW + sub;
        if (!pass_in_use<HD>(u, i, wave)) continue;
        float d = 1.0f;
        if (TYPE == G4_KV_Q8) {
            // as integers, magnitudes keep their order and infinities and NaN come last
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < M::VPL; k++) {
                const float e[4] = {x[i][k].x, x[i][k].y, x[i][k].z, x[i][k].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t b = __float_as_uint(e[j]) & 0x7fffffffu;
                    top = b > top ? b : top;
                }
            }
#pragma unroll
            for (int s = 1; s < M::LPR; s <<= 1) {
                const uint32_t o = __shfl_xor(top, s, 64);
                top = o > top ? o : top;
            }
            d = top < 0x7f800000u ? __uint_as_float(top) / 127.0f : __uint_as_float(0x7fc00000u);
            if (col == 0 && t >= u.t0 && t < u.t1)
                reinterpret_cast<float*>(pool + p.scale_off)[block * 16 + t] = d;
        }
#pragma unroll
        for (int k = 0; k < M::VPL; k++) {
            const float e[4] = {x[i][k].x, x[i][k].y, x[i][k].z, x[i][k].w};
            const int c = (k * M::LPR + col) * 4;
            T q[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float y = e[j];
                // d 0 or NaN: codes 0; past 127 only where d is subnormal
                if (TYPE == G4_KV_Q8) y = d > 0.0f ? fminf(fmaxf(rintf(y / d), -127.0f), 127.0f) : 0.0f;
                q[j] = Elem<TYPE>::of(y);
            }
            if (is_v) {
#pragma unroll
                for (int j = 0; j < 4; j++) *reinterpret_cast<T*>(img + kv_v_byte<ES>(t, c + j)) = q[j];
            } else {
                __builtin_memcpy(__builtin_assume_aligned(img + kv_k_byte<ES>(t, c), 4 * ES), q, 4 * ES);
            }
        }
    }
    lds_sync();
    uint8_t* out = pool + block * (16 * HD * ES);
    for (int x0 = tid; x0 < HD * ES; x0 += 256) {
        if (is_v) {
            const int t = (x0 >> 4 & 3) * 4;   // the piece's first token
            if (t >= u.t0 && t + 4 <= u.t1) {
                reinterpret_cast<uint4*>(out)[x0] = reinterpret_cast<const uint4*>(img)[x0];
            } else if (t < u.t1 && t + 4 > u.t0) {
                const T* from = reinterpret_cast<const T*>(img + x0 * 16);
                T* to = reinterpret_cast<T*>(out + x0 * 16);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (t + k >= u.t0 && t + k < u.t1) {
#pragma unroll
                        for (int j = 0; j < 4 / ES; j++) to[4 * j + k] = from[4 * j + k];
                    }
            }
        } else {
            const int t = x0 & 15;
            if (t >= u.t0 && t < u.t1) reinterpret_cast<uint4*>(out)[x0] = reinterpret_cast<const uint4*>(img)[x0];
        }
    }
}

}  // namespace
}  // namespace g4
