// attn_paged.hip -- attention of one new token of every sequence over the
// paged KV cache.
#include <math.h>

#include "g4_kvpage.h"
#include "g4_tile.h"

namespace g4 {
namespace {

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));

constexpr int kLgWG = 9, kPagedWG = 1 << kLgWG;   // workgroups that share the work, two a CU
constexpr int kHeadsWG = 16;                      // q heads of a workgroup: the columns of a product
constexpr float kLog2e = 1.4426950408889634f;

struct PagedArgs {
    KvPool p;
    const float* q;
    float* out;
    const int* lens;
    float* part;
    int q_stride, out_stride, n_seqs, window, n_heads;
    int group, ngrp;   // q heads a kv head, workgroup columns' groups of them
    int lead;          // units in front of an item's tiles
    int whole;         // 4, 8: a workgroup of so many waves an item, nothing to join; 0: split
    float scale;
};

// ---- shares of the work ------------------------------------------------------
// An item is a sequence, a kv head and up to 16 of its q heads; it consists of
// the 32-key tiles its window touches, behind lead units that stand for what
// it costs to begin and to end an item.  All items' units form one line,
// sequences in order, and workgroup w takes the units N w / 512 .. N (w + 1) /
// 512 - 1 of it, whatever the lengths are: a long sequence is spread over many
// workgroups, several short ones share one.  Without lead units a workgroup of
// short items outlives the others (the kernel, 64 sequences of 1 to 8192 keys,
// window 512, fp32: 35 us without, 17 with 3 of them, equal with 4, 31 with 1).
// One sequence has none: its items are alike, there is nothing to even out, and
// they would only give some workgroups a further round.  us with 0 / 3 lead
// units, both launches, 2 kv heads:
//   fp16 of 512: one sequence of 32768 keys 32 / 39, of 20000 27 / 27; two, four,
//   six, eight of 700 to 28000 38 / 28, 37 / 28, 71 / 67, 51 / 43; one of 20011
//   beside two of 700 31 / 27, beside eight 40 / 29;
//   bf16 of 256: one of 32768 beside 8, 24, 40, 100 of 10 to 300 26 / 23, 28 / 23,
//   35 / 27, 37 / 30; window 700, 8, 24, 40, 100 sequences 12 / 13, 18 / 15,
//   22 / 18, 34 / 33.
// Against it are a few sequences whose tiles divide by the workgroups by chance:
// fp16 of 512, two, four, eight of 32768 52 / 57, 104 / 113, 194 / 202, four of 2000
// 20 / 26, and one of nine batches of two to four ragged ones, 22 / 27.

// tiles of a sequence and its first one; 0 tiles: an empty sequence or a
// length that does not fit
__device__ __forceinline__ int seq_tiles(const PagedArgs& a, int len, int& first) {
    first = 0;
    if (len <= 0 || !a.p.fits(len)) return 0;
    if (a.window > 0 && len > a.window) first = (len - a.window) >> 5;
    return ((len - 1) >> 5) - first + 1;
}
__device__ __forceinline__ int seq_units(const PagedArgs& a, int len) {
    int first;
    const int t = seq_tiles(a, len, first);
    return t ? t + a.lead : 0;
}

// inclusive prefix sums over a wave: within rows of 16 by lane moves (lane -
// 1, 2, 4, 8, nothing from before the row), then the totals of the rows before
template <int CTRL>
__device__ __forceinline__ unsigned row_shr(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ unsigned wave_prefix(unsigned v) {
    v += row_shr<0x111>(v);
    v += row_shr<0x112>(v);
    v += row_shr<0x114>(v);
    v += row_shr<0x118>(v);
    auto at = [&](int l) { return (unsigned)__builtin_amdgcn_readlane((int)v, l); };
    const unsigned a = at(15), b = a + at(31), c = b + at(47), row = (threadIdx.x & 63) >> 4;
    return v + (row == 0 ? 0 : row == 1 ? a : row == 2 ? b : c);
}

struct Line {
    unsigned long long total;   // N, all units
    unsigned long long before;  // units of one (kv head, heads) before sequence s
    int s, len;
};

// N and the sequence that unit u = at(N) lies in (of_seq >= 0: that sequence
// instead), by the whole workgroup of 256 threads: a prefix sum over the
// lengths, which is cheaper than a launch that would leave it in memory.  Up
// to 64 sequences each wave finds it by itself.
template <typename At>
__device__ __forceinline__ Line find_line(const PagedArgs& a, At at, int of_seq, unsigned long long* red) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int rep = a.p.n_kv * a.ngrp;
    if (a.n_seqs <= 64) {
        const int len = lane < a.n_seqs ? a.lens[lane] : 0;
        const unsigned t = seq_units(a, len);   // 64 times 2^26 and less
        const unsigned x = wave_prefix(t);
        Line r;
        r.total = (unsigned long long)(unsigned)__builtin_amdgcn_readlane(x, 63) * rep;
        const unsigned long long u = at(r.total);
        const unsigned long long past = __ballot((unsigned long long)x * rep > u);
        r.s = of_seq >= 0 ? of_seq : past ? __builtin_ctzll(past) : 0;
        r.before = (unsigned)__builtin_amdgcn_readlane(x - t, r.s);
        r.len = __builtin_amdgcn_readlane(len, r.s);
        return r;
    }
    const int per = (a.n_seqs + 255) >> 8, s0 = tid * per;
    unsigned long long sum = 0;
    for (int i = 0; i < per; i++)
        if (s0 + i < a.n_seqs) sum += seq_units(a, a.lens[s0 + i]);
    unsigned long long x = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned long long o = __shfl_up(x, d, 64);
        if (lane >= d) x += o;
    }
    if (lane == 63) red[wave] = x;
    lds_sync();
    unsigned long long before = x - sum, all = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w < wave) before += red[w];
        all += red[w];
    }
    Line r;
    r.total = all * rep;
    const unsigned long long u = at(r.total);
    if (of_seq >= 0 ? s0 <= of_seq && of_seq < s0 + per : u >= before * rep && u < (before + sum) * rep) {
        int s = s0, len;
        for (;; s++) {
            len = a.lens[s];
            const int t = seq_units(a, len);
            if (of_seq >= 0 ? s == of_seq : u < (before + t) * rep) break;
            before += t;
        }
        red[4] = before;
        red[5] = (unsigned long long)(unsigned)s << 32 | (unsigned)len;
    }
    lds_sync();
    r.before = red[4];
    r.s = (int)(red[5] >> 32);
    r.len = (int)red[5];
    return r;
}

// the workgroup that has unit u of n: the quotient (u 512 + 511) / n, whose
// double is off by one at most
__device__ __forceinline__ int unit_wg(unsigned long long u, unsigned long long n) {
    unsigned long long w = (unsigned long long)(((double)u * kPagedWG + (kPagedWG - 1)) / (double)n);
    if ((n * w) >> kLgWG > u) w--;
    else if ((n * (w + 1)) >> kLgWG <= u) w++;
    return (int)w;
}

// floats of a partial result: [head][hd] sums, then each head's maximum and
// weight sum (16-byte aligned)
__host__ __device__ inline size_t part_floats(int group, int hd) {
    return ((size_t)(group < kHeadsWG ? group : kHeadsWG) * (hd + 2) + 3) & ~(size_t)3;
}

// ---- operands ------------------------------------------------------------------
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

template <int TYPE>
struct CacheType;
template <>
struct CacheType<G4_F32> { static constexpr int ES = 4, NT = 3; };
template <>
struct CacheType<G4_F16> { static constexpr int ES = 2, NT = 2; };   // 11 bits: two terms
template <>
struct CacheType<G4_BF16> { static constexpr int ES = 2, NT = 1; };
template <>
struct CacheType<G4_KV_Q8> { static constexpr int ES = 1, NT = 1; };

// two cached elements of a word pair as bf16 terms; codes (|c| <= 128) are exact in one
template <int TYPE>
__device__ __forceinline__ void pair_terms(const uint32_t* w, int i, uint32_t (&t)[CacheType<TYPE>::NT]) {
    if constexpr (TYPE == G4_F32) {
        split_pair<3>(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]), t);
    } else if constexpr (TYPE == G4_F16) {
        const h2_t h = bits_h2(w[i]);
        split_pair<2>((float)h[0], (float)h[1], t);
    } else if constexpr (TYPE == G4_BF16) {
        t[0] = w[i];
    } else {
        const int c0 = (int8_t)(w[i >> 1] >> (i & 1 ? 16 : 0)), c1 = (int8_t)(w[i >> 1] >> (i & 1 ? 24 : 8));
        t[0] = hi_halves(__float_as_uint((float)c0), __float_as_uint((float)c1));
    }
}
// eight elements that start at element 2 * i0 of w
template <int TYPE>
__device__ __forceinline__ void oct_terms(const uint32_t* w, int i0, b8_t (&t)[CacheType<TYPE>::NT]) {
    constexpr int NT = CacheType<TYPE>::NT;
    uint32_t p[4][NT];
#pragma unroll
    for (int i = 0; i < 4; i++) pair_terms<TYPE>(w, i0 + i, p[i]);
#pragma unroll
    for (int k = 0; k < NT; k++) t[k] = as_b8(p[0][k], p[1][k], p[2][k], p[3][k]);
}
// c + small += a . b over terms; what is left out is below 2^-30 of the
// product.  The leading terms' products have the sum c to themselves: a sum
// of 16 products and not of 16 x 6 loses that much less to rounding, which
// matters in scores (exponents), while the others are 2^-7 of it and less.
template <int NT>
__device__ __forceinline__ void mfma_terms(const b8_t (&a)[NT], const b8_t (&b)[3], f4_t& c, f4_t& small) {
#pragma unroll
    for (int i = NT - 1; i >= 0; i--)
#pragma unroll
        for (int j = 2; j >= 0; j--) {
            if (i + j == 0) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[0], c, 0, 0, 0);
            else if (i + j < 4) small = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], small, 0, 0, 0);
        }
}

// One wave takes 32 keys at a time, S^T = K Q^T (rows keys, columns q heads):
// a lane then holds the scores of one head at the eight keys 4 g + r and
// 16 + 4 g + r, which are, as they stand, its operand of O^T += V^T P^T (rows
// dims).  The cache's layout has each lane's K and V operands in 16
// consecutive bytes, so keys and values go from memory to the products through
// registers alone: no LDS, no barrier and no lane exchange but the one of the
// running maximum m.  It is put 2^8 above the largest score and moves only when
// one passes it, so that weights are at most 1 and their sums with V finite
// wherever the keys times the largest V are.  The q terms of a step come from
// LDS.  Bound by the cache's bytes where there are
// many: 40 sequences of 2000 to 30000 keys, 8 q heads on 2 kv heads of 256,
// bf16 150 us (5.4 TB/s; a plain read 6.25), fp32 5.4, codes 4.75; of 512, codes
// 5.0, fp32 4.9.  DEPTH loads of 1 KB are in flight a wave: 8, which one
// sequence of 200 keys out of HBM needs (bf16 of 256: 17 us with 4, 13 with 8,
// 12 with 16; of 512: 25 and 20), or 4 where 16-bit caches of 512 are split
// (fp16, one sequence of 32768 keys: 32 us with 4, 34 with 8).  More costs
// registers: codes of 512, 48 sequences, 155 us with 8, 215 with 16.
// WAVES 8: items taken whole, half the rounds
template <int TYPE, int HD, int DEPTH, int WAVES>
__global__ __launch_bounds__((64 * WAVES), 2) void attn_paged_kernel(PagedArgs a) {
    constexpr int ES = CacheType<TYPE>::ES, NT = CacheType<TYPE>::NT;
    constexpr int KC = HD * ES / 64;                      // 1 KB pieces of a 16-token block
    constexpr int CPS = ES == 4 ? 2 : 1;                  // pieces of a product step of 32 dims (ES 1: half a piece)
    constexpr int SPC = ES == 1 ? 2 : 1;                  // product steps of a piece
    constexpr int NL = 4 * KC, STEPS = HD / 32, NTILE = HD / 16, TPC = 4 / ES;   // TPC: 16-dim tiles of a V piece
    constexpr bool kKOnly = DEPTH <= 2 * KC;              // loads ahead of a tile's end are the next one's K
    static_assert(NL % DEPTH == 0, "ring");
    constexpr int kRounds = NTILE > 16 ? 2 : 1, NR = NTILE / kRounds;            // rounds of joining NR dim tiles,
    constexpr int NW = NR > WAVES ? NR / WAVES : 1;                              // NW of them a wave
    constexpr int kQBytes = STEPS * 3 * 1024, kSumBytes = WAVES * NR * 1024;
    __shared__ __align__(16) uint8_t buf[kQBytes > kSumBytes ? kQBytes : kSumBytes];
    __shared__ unsigned long long red[6];
    __shared__ float mls[2][WAVES][kHeadsWG];
    const bool items = WAVES == 8 || a.whole;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned w = blockIdx.x;
    const int rep = a.p.n_kv * a.ngrp;
    unsigned long long cur, end;
    int s, len, item, unit;
    // an item's q, 8 dims of a step and head a thread, on its way while the
    // pages are looked up where the registers allow it
    constexpr int QN = (STEPS + WAVES - 1) / WAVES;
    constexpr bool kEarlyQ = HD < 512 || (ES == 2 && DEPTH <= 4);
    float4 qx[QN][2];
    auto load_q = [&]() {
        const int kvh = item / a.ngrp, h0 = (item - kvh * a.ngrp) * kHeadsWG;
        const int nh = a.group - h0 < kHeadsWG ? a.group - h0 : kHeadsWG;
        const int h = kvh * a.group + h0 + (col < nh ? col : nh - 1);
        const float* qr = a.q + (size_t)s * a.q_stride + (size_t)h * HD;
#pragma unroll
        for (int i = 0; i < QN; i++) {
            const int st = STEPS % WAVES ? (i * WAVES + wave) % STEPS : i * WAVES + wave;
            const int d0 = ES == 4 ? st * 32 + g * 4 : ES == 2 ? st * 32 + g * 8 : (st >> 1) * 64 + g * 16 + (st & 1) * 8;
            qx[i][0] = *reinterpret_cast<const float4*>(qr + d0);
            qx[i][1] = *reinterpret_cast<const float4*>(qr + d0 + (ES == 4 ? 16 : 4));
        }
    };
    if (items) {
        s = (int)(w / (unsigned)rep);
        item = (int)w - s * rep;
        if (kEarlyQ) load_q();
        len = __builtin_amdgcn_readfirstlane(a.lens[s]);
        unit = 0;
        cur = 0;
        end = ~0ull;
    } else {
        const Line ln = find_line(a, [&](unsigned long long n) { return (n * w) >> kLgWG; }, -1, red);
        cur = (ln.total * w) >> kLgWG;
        end = (ln.total * (w + 1)) >> kLgWG;
        if (cur >= end) return;
        s = __builtin_amdgcn_readfirstlane(ln.s);
        len = __builtin_amdgcn_readfirstlane(ln.len);
        int f;
        const unsigned per = (unsigned)(seq_tiles(a, len, f) + a.lead);
        const unsigned long long off = cur - ln.before * rep;   // unit within the sequence's items
        item = __builtin_amdgcn_readfirstlane(off >> 32 ? (int)(off / per) : (int)((unsigned)off / per));
        unit = __builtin_amdgcn_readfirstlane((int)(off - (unsigned long long)item * per));
        if (kEarlyQ) load_q();
    }
    int first_tile, tiles = seq_tiles(a, len, first_tile);
    if (items && tiles == 0) {
        // no keys: zeros; a length that does not fit: NaN
        const float x = len == 0 ? 0.0f : __uint_as_float(0x7fc00000u);
        const int kvh = item / a.ngrp, hg = item - kvh * a.ngrp;
        const int nh = a.group - hg * kHeadsWG < kHeadsWG ? a.group - hg * kHeadsWG : kHeadsWG;
        float* to = a.out + (size_t)s * a.out_stride + (size_t)(kvh * a.group + hg * kHeadsWG) * HD;
        for (int i = tid; i < nh * HD / 4; i += 64 * WAVES) reinterpret_cast<float4*>(to)[i] = make_float4(x, x, x, x);
        return;
    }
    while (true) {
        const unsigned long long left = end - cur;
        const int unit1 = left < (unsigned long long)(tiles + a.lead - unit) ? unit + (int)left : tiles + a.lead;
        const int tile0 = unit > a.lead ? unit - a.lead : 0, tile1 = unit1 - a.lead;
        if (tile1 > tile0) {
            const int kvh = item / a.ngrp, hg = item - kvh * a.ngrp;
            const int nh = a.group - hg * kHeadsWG < kHeadsWG ? a.group - hg * kHeadsWG : kHeadsWG;
            const int head0 = kvh * a.group + hg * kHeadsWG;
            const int first = a.window > 0 && len > a.window ? len - a.window : 0;

            // ---- where a tile's two blocks are; one without a key in use is not read ----
            bool bad = false;
            auto pages = [&](int tile, bool on, int (&pg)[2]) {
                const int pos = (first_tile + tile) << 5;
                pg[0] = pg[1] = -1;
                if (on && first - pos < 16) {
                    pg[0] = __builtin_amdgcn_readfirstlane(a.p.page_of(s, pos));
                    bad = bad || pg[0] < 0;
                }
                if (on && len - pos > 16) {
                    pg[1] = __builtin_amdgcn_readfirstlane(a.p.page_of(s, pos + 16));
                    bad = bad || pg[1] < 0;
                }
            };
            auto block = [&](int tile, const int (&pg)[2], int i) {
                return a.p.block_of(pg[i] < 0 ? 0 : pg[i], kvh, ((first_tile + tile) << 5) + 16 * i);
            };
            auto rsrc = [&](const uint8_t* pool, int tile, const int (&pg)[2], __amdgpu_buffer_rsrc_t (&r)[2]) {
#pragma unroll
                for (int i = 0; i < 2; i++)
                    r[i] = __builtin_amdgcn_make_buffer_rsrc((void*)(pool + block(tile, pg, i) * (16 * HD * ES)), 0,
                                                             pg[i] < 0 ? 0 : 16 * HD * ES, kBufWord3);
            };
            // load i of a tile: K pieces in the order of the product steps, then V pieces, blocks in turn
            auto load = [&](int i, const __amdgpu_buffer_rsrc_t (&k)[2], const __amdgpu_buffer_rsrc_t (&v)[2]) {
                if (i < 2 * KC) {
                    const int b = i / CPS & 1, c = i / (2 * CPS) * CPS + i % CPS;
                    return buf_load16(k[b], lane * 16, c * 1024);
                }
                return buf_load16(v[i & 1], lane * 16, (i - 2 * KC) / 2 * 1024);
            };
            int tile = tile0 + wave, pg[2], npg[2];
            uint4 ring[DEPTH];
            __amdgpu_buffer_rsrc_t kr[2], vr[2], kn[2], vn[2];
            pages(tile, tile < tile1, pg);
            rsrc(a.p.kp, tile, pg, kr);
            rsrc(a.p.vp, tile, pg, vr);
#pragma unroll
            for (int i = 0; i < DEPTH; i++) ring[i] = load(i, kr, vr);

            // ---- q, times scale log2(e), as three terms in the products' order ----
            if (!kEarlyQ) load_q();
            const float qs = a.scale * kLog2e;
#pragma unroll
            for (int i = 0; i < QN; i++) {
                const int st = i * WAVES + wave;
                if (st >= STEPS) continue;
                float4 q0 = qx[i][0], q1 = qx[i][1];
                if (col >= nh) q0 = q1 = make_float4(0, 0, 0, 0);
                uint32_t t[4][3];
                split_pair<3>(q0.x * qs, q0.y * qs, t[0]);
                split_pair<3>(q0.z * qs, q0.w * qs, t[1]);
                split_pair<3>(q1.x * qs, q1.y * qs, t[2]);
                split_pair<3>(q1.z * qs, q1.w * qs, t[3]);
#pragma unroll
                for (int k = 0; k < 3; k++)
                    reinterpret_cast<uint4*>(buf)[(st * 3 + k) * 64 + lane] = make_uint4(t[0][k], t[1][k], t[2][k], t[3][k]);
            }
            lds_sync();

            // ---- the wave's tiles ----
            f4_t o[NTILE] = {};
            float m = -INFINITY, l = 0.0f;
            for (; tile < tile1; tile += WAVES) {
                // past the last tile the loads have no bytes to read
                pages(tile + WAVES, tile + WAVES < tile1, npg);
                if (!kKOnly) {
                    rsrc(a.p.kp, tile + WAVES, npg, kn);
                    rsrc(a.p.vp, tile + WAVES, npg, vn);
                }
                float ksc[8], vsc[8];
                if (TYPE == G4_KV_Q8) {
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const float4 x = reinterpret_cast<const float4*>(a.p.kp + a.p.scale_off)[block(tile, pg, b) * 4 + g];
                        const float4 y = reinterpret_cast<const float4*>(a.p.vp + a.p.scale_off)[block(tile, pg, b) * 4 + g];
                        ksc[4 * b] = x.x; ksc[4 * b + 1] = x.y; ksc[4 * b + 2] = x.z; ksc[4 * b + 3] = x.w;
                        vsc[4 * b] = y.x; vsc[4 * b + 1] = y.y; vsc[4 * b + 2] = y.z; vsc[4 * b + 3] = y.w;
                    }
                }
                auto take = [&](int i) {
                    const uint4 x = ring[i % DEPTH];
                    ring[i % DEPTH] = i + DEPTH < NL ? load(i + DEPTH, kr, vr) : load(i + DEPTH - NL, kn, vn);
                    return x;
                };
                f4_t sc[2] = {}, ss[2] = {};
                // q of a step is read while the one before it is worked on
                uint4 qn[SPC][3];
                auto read_q = [&](int st) {
#pragma unroll
                    for (int h = 0; h < SPC; h++)
#pragma unroll
                        for (int k = 0; k < 3; k++) qn[h][k] = reinterpret_cast<const uint4*>(buf)[((st * SPC + h) * 3 + k) * 64 + lane];
                };
                read_q(0);
#pragma unroll
                for (int st = 0; st < STEPS / SPC; st++) {
                    b8_t qt[SPC][3];
#pragma unroll
                    for (int h = 0; h < SPC; h++)
#pragma unroll
                        for (int k = 0; k < 3; k++) qt[h][k] = __builtin_bit_cast(b8_t, qn[h][k]);
                    if (st + 1 < STEPS / SPC) read_q(st + 1);
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        uint32_t x[4 * CPS];
#pragma unroll
                        for (int c = 0; c < CPS; c++) {
                            const uint4 y = take((st * 2 + b) * CPS + c);
                            x[4 * c] = y.x; x[4 * c + 1] = y.y; x[4 * c + 2] = y.z; x[4 * c + 3] = y.w;
                        }
#pragma unroll
                        for (int h = 0; h < SPC; h++) {
                            b8_t kt[NT];
                            oct_terms<TYPE>(x, 4 * h, kt);
                            mfma_terms<NT>(kt, qt[h], sc[b], ss[b]);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                // ---- weights ----
                const int pos = ((first_tile + tile) << 5) + 4 * g;
                float x[8], top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = pos + 16 * (i >> 2) + (i & 3);
                    float y = sc[i >> 2][i & 3] + ss[i >> 2][i & 3];
                    if (TYPE == G4_KV_Q8) y *= ksc[i];
                    x[i] = key >= first && key < len ? y : -INFINITY;
                    top = fmaxf(top, x[i]);
                }
                if (__any(top > m)) {
                    top = fmaxf(top, shfl_xor(top, 16));
                    top = fmaxf(top, shfl_xor(top, 32));
                    top = fmaxf(top + 8.0f, m);
                    const float f = top == m ? 1.0f : exp2f(m - top);
                    m = top;
                    l *= f;
#pragma unroll
                    for (int i = 0; i < NTILE; i++) o[i] *= f;
                }
                uint32_t pw[4][3];
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    float p[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int key = pos + 16 * ((i + j) >> 2) + ((i + j) & 3);
                        const bool in = key >= first && key < len;
                        p[j] = in ? exp2f(x[i + j] - m) : 0.0f;
                        l += p[j];
                        if (TYPE == G4_KV_Q8) p[j] = in ? p[j] * vsc[i + j] : 0.0f;
                    }
                    split_pair<3>(p[0], p[1], pw[i / 2]);
                }
                b8_t pt[3];
#pragma unroll
                for (int k = 0; k < 3; k++) pt[k] = as_b8(pw[0][k], pw[1][k], pw[2][k], pw[3][k]);
                // elements of keys not in use count as 0, whatever is left there
                uint32_t keep[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = pos + 16 * (i >> 2) + (i & 3);
                    keep[i] = key >= first && key < len ? 0xffffffffu : 0u;
                }
                if (kKOnly) rsrc(a.p.kp, tile + WAVES, npg, kn);
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    uint4 y[2];
                    y[0] = take(2 * KC + 2 * c);
                    y[1] = take(2 * KC + 2 * c + 1);
#pragma unroll
                    for (int i = 0; i < TPC; i++) {
                        // this lane's dim of tile c * TPC + i at its eight keys
                        uint32_t v[2 * ES];
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            const uint32_t z[4] = {y[b].x, y[b].y, y[b].z, y[b].w};
#pragma unroll
                            for (int j = 0; j < ES; j++) {
                                uint32_t k;
                                if (ES == 4) k = keep[4 * b + j];
                                else if (ES == 2) k = __builtin_amdgcn_perm(keep[4 * b + 2 * j + 1], keep[4 * b + 2 * j], 0x05040100u);
                                else k = __builtin_amdgcn_perm(__builtin_amdgcn_perm(keep[4 * b + 3], keep[4 * b + 2], 0x0c0c0400u),
                                                               __builtin_amdgcn_perm(keep[4 * b + 1], keep[4 * b], 0x0c0c0400u), 0x05040100u);
                                v[b * ES + j] = z[i * ES + j] & k;
                            }
                        }
                        b8_t vt[NT];
                        oct_terms<TYPE>(v, 0, vt);
                        mfma_terms<NT>(vt, pt, o[c * TPC + i], o[c * TPC + i]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (kKOnly) rsrc(a.p.vp, tile + WAVES, npg, vn);
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    kr[b] = kn[b];
                    vr[b] = vn[b];
                    pg[b] = npg[b];
                }
            }

            // ---- the waves' sums, a part of the dims by each (one wave after another,
            // bf16 of 256, one sequence of 203 keys: 8.7 -> 8.0 us with q's loads ahead) ----
            l += shfl_xor(l, 16);
            l += shfl_xor(l, 32);
            if (bad) l = __uint_as_float(0x7fc00000u);
            const bool whole = tile0 == 0 && tile1 == tiles;
            float* slot = a.part + ((size_t)w * 2 + (tile0 == 0)) * part_floats(a.group, HD);
            float* to = whole ? a.out + (size_t)s * a.out_stride + (size_t)(head0 + col) * HD : slot + col * HD;
            float* stats = slot + (a.group < kHeadsWG ? a.group : kHeadsWG) * HD + 2 * col;
            if (tile1 - tile0 == 1) {   // wave 0 had the only tile
                if (wave == 0 && col < nh) {
                    const float f = whole ? 1.0f / l : 1.0f;
#pragma unroll
                    for (int i = 0; i < NTILE; i++) {
                        const f4_t r = o[i] * f;
                        *reinterpret_cast<f4_t*>(to + i * 16 + g * 4) = r;
                    }
                    if (!whole && g == 0) *reinterpret_cast<float2*>(stats) = make_float2(m, l);
                }
            } else {
                if (g == 0) {
                    mls[0][wave][col] = m;
                    mls[1][wave][col] = l;
                }
                lds_sync();   // q is no longer needed
                f4_t* box = reinterpret_cast<f4_t*>(buf) + lane;
                float f[WAVES], top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int r = 0; r < kRounds; r++) {
                    if (r) lds_sync();
#pragma unroll
                    for (int i = 0; i < NR; i++) box[(wave * NR + i) * 64] = o[r * NR + i];
                    if (r == 0) {
#pragma unroll
                        for (int i = 0; i < WAVES; i++) top = fmaxf(top, f[i] = mls[0][i][col]);
#pragma unroll
                        for (int i = 0; i < WAVES; i++) {
                            f[i] = f[i] == top ? 1.0f : exp2f(f[i] - top);
                            sum += f[i] * mls[1][i][col];
                        }
                        if (!whole && wave == 0 && g == 0 && col < nh) *reinterpret_cast<float2*>(stats) = make_float2(top, sum);
                        const float x = whole ? 1.0f / sum : 1.0f;
#pragma unroll
                        for (int i = 0; i < WAVES; i++) f[i] *= x;
                    }
                    lds_sync();
#pragma unroll
                    for (int i = 0; i < NW; i++) {
                        const int t = wave * NW + i;
                        if (t >= NR) break;
                        f4_t y = box[t * 64] * f[0];
#pragma unroll
                        for (int k = 1; k < WAVES; k++) y += box[(k * NR + t) * 64] * f[k];
                        if (col < nh) *reinterpret_cast<f4_t*>(to + (r * NR + t) * 16 + g * 4) = y;
                    }
                }
            }
            lds_sync();   // the sums' place takes q again
        }
        cur += (unsigned)(unit1 - unit);
        if (items || cur >= end) break;
        unit = 0;
        if (++item == rep) {
            item = 0;
            do {
                len = __builtin_amdgcn_readfirstlane(a.lens[++s]);
                tiles = seq_tiles(a, len, first_tile);
            } while (tiles == 0);
        }
        if (kEarlyQ) load_q();
    }
}

// Joins the pieces of every sequence and head that more than one workgroup
// took, with the weights 2^(m_i - max m); sequences without keys get zeros,
// those whose length does not fit NaN.  Latency: 4.3 to 6 us, of which the
// launch, the lengths, the pieces' maxima and their sums are a chain.
// D of the HD dims a workgroup (blockIdx.z): 64 where there are few heads and
// sequences, whose pieces then are as many.
template <int HD, int D>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(PagedArgs a) {
    constexpr int LPR = D / 4, GR = 256 / LPR;   // lanes a row of D floats, pieces at a time
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int kvh = h / a.group, hg = (h - kvh * a.group) / kHeadsWG, col = h - kvh * a.group - hg * kHeadsWG;
    __shared__ unsigned long long red[6];
    __shared__ float fac[kPagedWG], wred[4];
    __shared__ __align__(16) float4 acc[256];
    float* out = a.out + (size_t)s * a.out_stride + (size_t)h * HD + blockIdx.z * D;
    const int len = a.lens[s];
    int first;
    const int tiles = seq_tiles(a, len, first);
    if (tiles == 0) {
        const float x = len == 0 ? 0.0f : __uint_as_float(0x7fc00000u);
        if (tid < LPR) reinterpret_cast<float4*>(out)[tid] = make_float4(x, x, x, x);
        return;
    }
    const Line ln = find_line(a, [](unsigned long long) { return 0ull; }, s, red);
    const unsigned long long n = ln.total;
    const unsigned long long u0 =
        ln.before * (a.p.n_kv * a.ngrp) + (unsigned long long)(kvh * a.ngrp + hg) * (tiles + a.lead) + a.lead;
    const int w0 = unit_wg(u0, n), w1 = unit_wg(u0 + tiles - 1, n);
    if (w0 == w1) return;   // one workgroup had it all
    // fewer units than workgroups: a unit each, some workgroups between them without one
    const bool few = n < kPagedWG;
    const int np = few ? tiles : w1 - w0 + 1, gh = a.group < kHeadsWG ? a.group : kHeadsWG;
    const size_t pf = part_floats(a.group, HD);
    auto slot = [&](int i) { return a.part + ((size_t)(few ? unit_wg(u0 + i, n) : w0 + i) * 2 + (i == 0)) * pf; };
    // the first pieces' sums are on their way while the factors are found
    const int c = tid % LPR, gr = tid / LPR;
    auto sums = [&](int i, float4 (&y)[8]) {
#pragma unroll
        for (int k = 0; k < 8; k++)
            y[k] = reinterpret_cast<const float4*>(slot(i + k * GR < np ? i + k * GR : 0) + col * HD + blockIdx.z * D)[c];
    };
    float4 y[8];
    sums(gr, y);
    // maxima, factors, weight sums: pieces tid and tid + 256
    float m[2], l[2], top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int i = tid + 256 * k;
        m[k] = -INFINITY;
        l[k] = 0.0f;
        if (i < np) {
            const float2 x = reinterpret_cast<const float2*>(slot(i) + gh * HD)[col];
            m[k] = x.x;
            l[k] = x.y;
        }
        top = fmaxf(top, m[k]);
    }
    top = wave_max(top);
    if ((tid & 63) == 0) wred[tid >> 6] = top;
    lds_sync();
    top = fmaxf(fmaxf(wred[0], wred[1]), fmaxf(wred[2], wred[3]));
    lds_sync();
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const float f = m[k] == top ? 1.0f : exp2f(m[k] - top);
        fac[tid + 256 * k] = f;
        sum += f * l[k];
    }
    sum = wave_sum(sum);
    if ((tid & 63) == 0) wred[tid >> 6] = sum;
    lds_sync();
    sum = (wred[0] + wred[1]) + (wred[2] + wred[3]);
    float4 x = make_float4(0, 0, 0, 0);
    for (int i = gr; i < np; i += 8 * GR) {
        if (i > gr) sums(i, y);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (i + k * GR >= np) continue;
            const float f = fac[i + k * GR];
            x.x = __builtin_fmaf(f, y[k].x, x.x);
            x.y = __builtin_fmaf(f, y[k].y, x.y);
            x.z = __builtin_fmaf(f, y[k].z, x.z);
            x.w = __builtin_fmaf(f, y[k].w, x.w);
        }
    }
    acc[tid] = x;
    lds_sync();
    if (tid < LPR) {
#pragma unroll
        for (int k = 1; k < GR; k++) {
            const float4 y = acc[k * LPR + tid];
            x.x += y.x;
            x.y += y.y;
            x.z += y.z;
            x.w += y.w;
        }
        const float r = 1.0f / sum;
        reinterpret_cast<float4*>(out)[tid] = make_float4(x.x * r, x.y * r, x.z * r, x.w * r);
    }
}

// keys up to which a workgroup takes an item whole (figures: g4_attn_decode_paged),
// and those of a round of four waves, past which it has eight
constexpr int kRound = 128;
constexpr int whole_keys(int type, int hd) {
    const int cap = type == G4_F32 ? 256 : 512, fit = (type == G4_F32 ? 65536 : 131072) / hd;
    return fit < cap ? fit : cap;
}

template <int TYPE, int HD>
void launch_paged(const PagedArgs& a) {
    constexpr int ES = CacheType<TYPE>::ES, NL = HD * ES / 16, W = NL < 8 ? NL : 8, D = ES == 2 && HD == 512 ? 4 : W;
    if (a.whole) {
        const int items = a.n_seqs * a.p.n_kv * a.ngrp;
        if constexpr (whole_keys(TYPE, HD) > kRound) {
            if (a.whole == 8) {
                hipLaunchKernelGGL((attn_paged_kernel<TYPE, HD, W, 8>), dim3(items), dim3(512), 0, g4_stream(), a);
                return;
            }
        }
        hipLaunchKernelGGL((attn_paged_kernel<TYPE, HD, W, 4>), dim3(items), dim3(256), 0, g4_stream(), a);
        return;
    }
    hipLaunchKernelGGL((attn_paged_kernel<TYPE, HD, D, 4>), dim3(kPagedWG), dim3(256), 0, g4_stream(), a);
    if (a.n_heads * a.n_seqs < 256)
        hipLaunchKernelGGL((attn_paged_join_kernel<HD, 64>), dim3(a.n_heads, a.n_seqs, HD / 64), dim3(256), 0, g4_stream(), a);
    else
        hipLaunchKernelGGL((attn_paged_join_kernel<HD, HD>), dim3(a.n_heads, a.n_seqs, 1), dim3(256), 0, g4_stream(), a);
}
template <int TYPE>
void launch_paged(const PagedArgs& a, int hd) {
    if (hd == 64) launch_paged<TYPE, 64>(a);
    else if (hd == 128) launch_paged<TYPE, 128>(a);
    else if (hd == 256) launch_paged<TYPE, 256>(a);
    else launch_paged<TYPE, 512>(a);
}

}  // namespace
}  // namespace g4

using namespace g4;

extern "C" size_t g4_attn_decode_paged_part_bytes(int n_heads, int n_kv, int hd) {
    if (n_heads < 1 || n_kv < 1 || n_heads % n_kv || (hd != 64 && hd != 128 && hd != 256 && hd != 512)) return 0;
    return (size_t)kPagedWG * 2 * part_floats(n_heads / n_kv, hd) * 4;
}

extern "C" int g4_attn_decode_paged(const float* q, int q_stride, const void* kp, const void* vp, int type, int n_pages,
                                    int page, int n_kv, int hd, const int* table, int table_stride, const int* lens,
                                    int n_seqs, int window, int n_heads, float attn_scale, float* part, float* out,
                                    int out_stride) {
    const char* who = "g4_attn_decode_paged";
    PagedArgs a = {};
    const int rc = kv_pool_check(who, &a.p, kp, vp, type, n_pages, page, n_kv, hd, table, table_stride);
    if (rc) return rc;
    G4_CHECK_ARG(n_heads > 0 && n_heads <= 65535 && n_heads % n_kv == 0, "%s: %d heads over %d kv heads", who, n_heads, n_kv);
    G4_CHECK_ARG(q && lens && part && out && al16(q) && al16(part) && al16(out), "%s: null or unaligned pointer", who);
    G4_CHECK_ARG(q_stride % 4 == 0 && q_stride / hd >= n_heads && out_stride % 4 == 0 && out_stride / hd >= n_heads,
                 "%s: strides %d, %d (multiples of 4, n_heads * hd at least)", who, q_stride, out_stride);
    G4_CHECK_ARG(n_seqs > 0 && n_seqs <= kKvMaxSeqs && window >= 0, "%s: %d sequences (1 to %d), window %d", who, n_seqs,
                 kKvMaxSeqs, window);
    a.q = q; a.out = out; a.lens = lens; a.part = part; a.q_stride = q_stride; a.out_stride = out_stride;
    a.n_seqs = n_seqs; a.window = window; a.n_heads = n_heads; a.scale = attn_scale;
    a.group = n_heads / n_kv;
    a.ngrp = (a.group + kHeadsWG - 1) / kHeadsWG;
    a.lead = n_seqs > 1 ? 3 : 0;
    // Where a sequence cannot have more keys to look at than that, by its table
    // or the window, a workgroup takes an item whole and there is nothing to
    // join: some rounds of its waves cost less than the second launch.
    // head_dim 256, 2 kv heads, 1 / 64 / 200 sequences: bf16, 250 keys 6.8 / 7.8
    // / 19.7 us whole, 11.2 / 15.0 / 30.5 split, 500 keys 9.1 / 18.4 / 37.5 and
    // 11.5 / 19.7 / 43.8; codes, 500 keys 11.5 / 12.4 / 22.0 and 12.1 / 17.4 / 34.7;
    // fp32, 250 keys 11.8 / 18.1 / 41 and 14.8 / 21.2 / 48.2.  Of 512: bf16, 250
    // keys 10.5 and 13.9 (one); fp32, 120 keys 16.8 and 21.0, 250 keys with four
    // waves 26.3 and 21.3.  Eight waves where each such workgroup has a CU and more
    // than a round of four to do: against four, one sequence of 250 keys 6.8
    // and 7.6 us in bf16, 11.8 and 15.5 in fp32; 64 of 500 keys 18.4 and 17.1.
    long most = (long)table_stride * page;
    if (window > 0 && window < most) most = window;
    const size_t items = (size_t)n_seqs * n_kv * a.ngrp;
    a.whole = most > whole_keys(type, hd) || !kv_grid_fits(items, 256) ? 0 : items <= 256 && most > kRound ? 8 : 4;
    if (type == G4_F32) launch_paged<G4_F32>(a, hd);
    else if (type == G4_F16) launch_paged<G4_F16>(a, hd);
    else if (type == G4_BF16) launch_paged<G4_BF16>(a, hd);
    else launch_paged<G4_KV_Q8>(a, hd);
    return g4_check_launch("attn_paged_kernel");
}
