// attn_packed.hip -- causal attention of whole prompts, packed one after the
// other.
//
// Two launches.  The first puts K and V of every sequence into blocks of 32
// keys in the order in which the matrix cores take them (32 x 32 x 16
// products, whole kilobytes of 64 lanes x 16 bytes), a sequence's blocks
// padded with zeros:
//   K (operand rows = keys): lane 32 h + t of piece s holds key t's dims
//     16 s + 8 h .. + 7;
//   V (operand rows = dims): lane 32 h + n of piece 2 c + t holds dim 32 c + n
//     of keys 16 t + 8 (j / 4) + 4 h + j % 4, j = 0 .. 7: the keys whose
//     scores the lane half gets out of the first product.
// The second launch then needs no transpose, no bank-conflict pattern and no
// care for a neighbour's rows: tiles go from memory to LDS as they are
// (buffer loads to LDS) and from there to the operands.
//
// A row of K or V that holds an infinity or NaN is stored as zeros and marked:
// a query that sees it gets the score NaN there, others never meet it.
#include <atomic>

#include "g4_attn_tile.h"
#include "g4_kvpage.h"

namespace g4 {
namespace {

struct PackedArgs {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    uint8_t* work;
    const int* cu;
    int q_stride, kv_stride, out_stride, n_seqs, m, window, n_heads, n_kv, group;
    int extra;      // units a sequence may need beyond its share
    float scale;
};

// fp32 operands are products of three pairs of fp16 halves of a scaled row:
// x = 2^e (hi + lo), the row's largest |hi| in [2^14, 2^15], so that x is met
// within 2^-22 of itself or 2^-39 of the row's largest.
template <int T>
struct Kind;
template <>
struct Kind<G4_F32> {
    static constexpr int ES = 4, NS = 2;
    typedef float t;
    typedef h8_t op;
};
template <>
struct Kind<G4_F16> {
    static constexpr int ES = 2, NS = 1;
    typedef _Float16 t;
    typedef h8_t op;
};
template <>
struct Kind<G4_BF16> {
    static constexpr int ES = 2, NS = 1;
    typedef __bf16 t;
    typedef b8_t op;
};
// A block: K pieces (fp32: hi, then lo), V pieces (likewise), then 512 bytes:
// fp32: each key's K scale 2^e, V exponent e, 2^-e; the masks of marked keys (K, V);
// fp32: the weight sum below which lost_weight is asked for.
constexpr int kMeta = 512, kMetaVExp = 128, kMetaVInv = 256, kMetaMask = 384, kMetaLost = 392;
__host__ __device__ constexpr size_t block_bytes(int hd, int es) { return (size_t)64 * hd * es + kMeta; }

// ---- first launch: K and V into blocks -----------------------------------------
// blockIdx: block, kv head, K or V.  Sequence s has the blocks (cu[s] >> 5) + s
// and on.  Bytes and latency (the starts, the rows, the stores are a chain):
// 8191 rows of 2 x 256 in bf16 9.4 us (3.6 TB/s read and written), 7022 of 2 x
// 512 in fp32 26 us (4.4).
template <int T, int HD>
__global__ __launch_bounds__(256) void packed_layout_kernel(PackedArgs a) {
    typedef typename Kind<T>::t E;
    constexpr int ES = Kind<T>::ES, NS = Kind<T>::NS;
    constexpr int VW = 16 / ES;                            // elements of a 16-byte load
    constexpr int LPR = HD / VW < 64 ? HD / VW : 64;       // lanes a row
    constexpr int VPL = HD / VW / LPR, RPW = 64 / LPR, PASS = 8 / RPW;
    __shared__ __align__(16) uint8_t img[64 * HD];         // one half (hi or lo) of K or V
    __shared__ unsigned marks;
    __shared__ int lowest;                                 // V: smallest exponent of the rows there are
    const unsigned id = blockIdx.x;
    const SeqAt sq = find_seq(a.cu, nullptr, a.n_seqs, 1, 5, 1, id);
    const int r0 = sq.r0, r1 = sq.r1;
    const unsigned b = id - (((unsigned)r0 >> 5) + (unsigned)sq.s);
    if (r0 < 0 || r1 <= r0 || r1 > a.m || b >= (unsigned)((r1 - r0 + 31) >> 5)) return;
    const int row0 = r0 + (int)b * 32, rows = r1 - row0 < 32 ? r1 - row0 : 32;
    const bool is_v = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int sub = lane / LPR, col = lane % LPR;
    // V: a thread has G keys next to each other, which it writes at once (one at
    // a time: 9.9 and 27.5 us)
    constexpr int G = PASS < 4 ? PASS : 4;
    auto key = [&](int i) { return is_v ? (wave * RPW + sub) * PASS + i : (i * 4 + wave) * RPW + sub; };
    // LDS slot of lane l's 16 bytes of a piece: the lanes of a row write to
    // one slot of many pieces (K) or to every 4th or 8th slot (V), all on the
    // same banks without the exchange
    auto swz = [&](int piece, int l) {
        return piece * 64 + (is_v ? l ^ (l >> 3 & 3) ^ (piece >> 1 & 1) ^ (piece & 4) : l ^ ((piece * 2 + (l >> 5)) & 7));
    };
    const E* src = (const E*)(is_v ? a.v : a.k) + (size_t)blockIdx.y * HD;
    if (tid == 0) {
        marks = 0;
        lowest = 113;
    }
    uint4 x[PASS][VPL];
#pragma unroll
    for (int i = 0; i < PASS; i++) {
        const int t = key(i);
        const size_t r = row0 + (t < rows ? t : 0);
#pragma unroll
        for (int k = 0; k < VPL; k++)
            x[i][k] = *reinterpret_cast<const uint4*>(src + r * a.kv_stride + (k * LPR + col) * VW);
    }
    lds_sync();
    uint8_t* rec = a.work + ((size_t)id * a.n_kv + blockIdx.y) * block_bytes(HD, ES);
    uint8_t* out = rec + (is_v ? 32 * HD * ES : 0);
    float* meta = reinterpret_cast<float*>(rec + 64 * HD * ES);
    float sc[PASS];
#pragma unroll
    for (int i = 0; i < PASS; i++) {
        const int t = key(i);
        // the row's largest magnitude, as integers: infinities and NaN come last
        unsigned top = 0;
#pragma unroll
        for (int k = 0; k < VPL; k++) {
            const unsigned w[4] = {x[i][k].x, x[i][k].y, x[i][k].z, x[i][k].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                unsigned m;
                if (ES == 4) m = w[j] & 0x7fffffffu;
                else m = (w[j] & 0x7fffu) > (w[j] >> 16 & 0x7fffu) ? w[j] & 0x7fffu : w[j] >> 16 & 0x7fffu;
                top = m > top ? m : top;
            }
        }
#pragma unroll
        for (int d = 1; d < LPR; d <<= 1) {
            const unsigned o = __shfl_xor(top, d, 64);
            top = o > top ? o : top;
        }
        const bool finite = top < (T == G4_F32 ? 0x7f800000u : T == G4_F16 ? 0x7c00u : 0x7f80u);
        if (t >= rows || !finite) {
#pragma unroll
            for (int k = 0; k < VPL; k++) x[i][k] = make_uint4(0, 0, 0, 0);
        }
        if (t < rows && !finite && col == 0) atomicOr(&marks, 1u << t);
        sc[i] = 1.0f;
        if (T == G4_F32) {
            const int low = is_v ? kLowV : kLowK;
            const int e = t < rows && finite && (int)(top >> 23) > low ? (int)(top >> 23) : low;
            sc[i] = row_scale(e);
            if (col == 0) {
                if (is_v) {
                    meta[kMetaVExp / 4 + t] = (float)(e - 141);
                    meta[kMetaVInv / 4 + t] = sc[i];
                    if (t < rows && finite) atomicMin(&lowest, e - 141);
                } else {
                    meta[t] = row_scale_inv(e);
                }
            }
        }
    }
    // VW halves (hi or lo) of a thread's row i, dims c ..
    auto halves = [&](int i, int k, int half, uint16_t (&e)[VW]) {
        const unsigned w[4] = {x[i][k].x, x[i][k].y, x[i][k].z, x[i][k].w};
        if constexpr (T == G4_F32) {
#pragma unroll
            for (int j = 0; j < VW; j += 2) {
                h2v_t hi, lo;
                split2(__uint_as_float(w[j]), __uint_as_float(w[j + 1]), sc[i], hi, lo);
                const unsigned y = __builtin_bit_cast(unsigned, half ? lo : hi);
                e[j] = (uint16_t)y;
                e[j + 1] = (uint16_t)(y >> 16);
            }
        } else {
            __builtin_memcpy(e, w, 16);
        }
    };
#pragma unroll
    for (int half = 0; half < NS; half++) {
        if (half) lds_sync();   // the first half has been read
        if (is_v) {
#pragma unroll
            for (int i = 0; i < PASS; i += G)
#pragma unroll
                for (int k = 0; k < VPL; k++) {
                    uint16_t e[G][VW];
#pragma unroll
                    for (int r = 0; r < G; r++) halves(i + r, k, half, e[r]);
                    // key t = 16 u + 8 b + 4 h + r
                    const int t = key(i), c = (k * LPR + col) * VW;
                    const int u = t >> 4, h = t >> 2 & 1, slot = (t >> 3 & 1) * 4 + (t & 3);
#pragma unroll
                    for (int j = 0; j < VW; j++) {
                        const int d = c + j;
                        uint16_t y[G];
#pragma unroll
                        for (int r = 0; r < G; r++) y[r] = e[r][j];
                        __builtin_memcpy(__builtin_assume_aligned(img + swz((d >> 5) * 2 + u, h * 32 + (d & 31)) * 16 + slot * 2, G * 2),
                                         y, G * 2);
                    }
                }
        } else {
#pragma unroll
            for (int i = 0; i < PASS; i++)
#pragma unroll
                for (int k = 0; k < VPL; k++) {
                    const int t = key(i), c = (k * LPR + col) * VW;
                    uint16_t e[VW];
                    halves(i, k, half, e);
                    __builtin_memcpy(__builtin_assume_aligned(img + swz(c >> 4, (c >> 3 & 1) * 32 + t) * 16 + (c & 7) * 2, VW * 2), e,
                                     VW * 2);
                }
        }
        lds_sync();
        for (int i = tid; i < 4 * HD; i += 256)
            reinterpret_cast<uint4*>(out + half * 64 * HD)[i] = reinterpret_cast<const uint4*>(img)[swz(i >> 6, i & 63)];
    }
    if (tid == 0) {
        reinterpret_cast<unsigned*>(meta)[kMetaMask / 4 + is_v] = marks;
        if (T == G4_F32 && is_v) meta[kMetaLost / 4] = __builtin_ldexpf(1.0f, 48 - 126 - lowest);
    }
}

// ---- few rows: one launch, fp32 throughout --------------------------------------
// A workgroup a row and head, a wave a few keys at a time (one: 64 rows of 256
// 6.4 us against 5.2; four q heads of a kv head together, 7.9): a hundredth of
// the products' rate, without the latency of a second launch and of tiles.
// Taken where rows x keys x heads cannot pass 2^18 however the rows fall into
// sequences.  One sequence, 8 heads, fp32 / bf16, this against the other: 128
// rows of 256 12.3 / 13.3 against 24.2 / 15.0 us, 192 rows 18.2 / 19.4 against
// 28.7 / 16.6, 256 rows 38 / 42 against 33 / 18.7; 128 rows of 512 20.6 / 16.0
// against 30.3 / 20.9.
constexpr double kFewPairs = 1 << 18;
template <int T, int HD>
__global__ __launch_bounds__(256) void attn_packed_few_kernel(PackedArgs a) {
    typedef typename Kind<T>::t E;
    constexpr int N = HD / 64, KB = N * sizeof(E) <= 16 ? 4 : 2;   // a lane's dims; keys at a time
    struct alignas(N * sizeof(E) < 16 ? N * sizeof(E) : 16) Dims {
        E x[N];
    };
    const int row = blockIdx.x, h = blockIdx.y, kvh = h / a.group;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float red[4][HD + 2];
    const SeqAt sq = find_seq(a.cu, nullptr, a.n_seqs, 1, 0, 0, (unsigned)row);
    const int r0 = sq.r0, r1 = sq.r1;
    if (r0 < 0 || r1 > a.m || row < r0 || row >= r1) return;
    const int first = a.window > 0 && row - r0 >= a.window ? row + 1 - a.window : r0;
    auto dims = [&](const void* x, int stride, int r, int head) {
        return reinterpret_cast<const Dims*>((const E*)x + (size_t)r * stride + (size_t)head * HD)[lane];
    };
    const Dims qx = dims(a.q, a.q_stride, row, h);
    float q[N], o[N] = {}, m = -FLT_MAX, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) q[i] = (float)qx.x[i] * (a.scale * kLog2e);
    for (int t0 = first + wave * KB; t0 <= row; t0 += 4 * KB) {
        Dims k[KB], v[KB];
#pragma unroll
        for (int j = 0; j < KB; j++) {
            const int t = t0 + j <= row ? t0 + j : row;
            k[j] = dims(a.k, a.kv_stride, t, kvh);
            v[j] = dims(a.v, a.kv_stride, t, kvh);
        }
        float x[KB], mn = m;
#pragma unroll
        for (int j = 0; j < KB; j++) {
            x[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < N; i++) x[j] = __builtin_fmaf(q[i], (float)k[j].x[i], x[j]);
            x[j] = wave_sum(x[j]);
            if (t0 + j > row) x[j] = -INFINITY;
            mn = fmaxf(mn, x[j]);
        }
        const float f = exp2f(m - mn);
        l *= f;
        m = mn;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] *= f;
#pragma unroll
        for (int j = 0; j < KB; j++) {
            const float w = exp2f(x[j] - mn);
            l += w;
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = __builtin_fmaf(w, (float)v[j].x[i], o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) red[wave][lane * N + i] = o[i];
    if (lane == 0) {
        red[wave][HD] = m;
        red[wave][HD + 1] = l;
    }
    lds_sync();
    float top = red[0][HD], f[4], den = 0.0f;
#pragma unroll
    for (int w = 1; w < 4; w++) top = fmaxf(top, red[w][HD]);
#pragma unroll
    for (int w = 0; w < 4; w++) {
        f[w] = exp2f(red[w][HD] - top);
        den += f[w] * red[w][HD + 1];
    }
    E* out = (E*)a.out + (size_t)row * a.out_stride + (size_t)h * HD;
    for (int d = threadIdx.x; d < HD; d += 256) {
        float num = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) num += f[w] * red[w][d];
        out[d] = (E)(num / den);
    }
}

// ---- second launch ------------------------------------------------------------------
// A wave's job is 32 rows of one q head; a workgroup takes NJ consecutive jobs
// of a kv head (the heads of 32 rows, then the next 32 rows), which share its
// tiles of 32 keys in LDS.  S^T = K Q^T (rows keys, columns q rows): a lane
// holds 16 of a row's 32 scores, which are, as they stand, its operand of
// O^T += V^T P^T.  The running maximum moves only when a score passes it (bf16,
// where it stands 2^8 above the largest; fp16, fp32: by 2^8, 2^4).  DS 2
// (head_dim 512, whose q and o would not fit a wave's registers): a job's dims
// are halved over two waves, whose partial scores meet in LDS; K and V of a tile
// have one place each, and the next tile's K is on its way while V is worked on,
// and the other way round.
// KSP 2 (16 bits): the two waves of a SIMD are given the same job and every
// other tile, so that there are twice the workgroups, half as long, and the
// one does its second product while the other is at its weights: waves 4 .. 7
// put it off to the next tile.  Their sums meet at the end, in LDS.  (8191 rows
// in bf16, 8 heads of 256: 404 us with eight jobs a workgroup in step, 333 so.)
// What bounds it: the matrix cores under the card's power limit.  Four prompts
// of 4096 rows, 8 heads of 256 (128: 32): bf16 293-370 us from card to card,
// 745-940 TFLOP/s at 1.75-2.1 GHz where an 8192^3 library product reaches 1182;
// fp32 815-900 us, 305-337 TFLOP/s and three times as many products.  Copies to
// LDS alone (55 bytes/ns a CU) would take 155 and 305 us.  Three independent
// sums instead of two, the next tile's scores computed beside this tile's
// weights and wave priorities around the products changed nothing or lost.
template <int T, int HD>
struct Plan {
    static constexpr int ES = Kind<T>::ES;
    static constexpr int DS = HD == 512 ? 2 : 1;                     // fp32 at 512: attn_packed_wide_kernel
    static constexpr int NW = T == G4_F32 ? 4 : 8;                   // waves; 8: two a SIMD
    static constexpr int KSP = NW == 8 && DS == 1 ? 2 : 1;           // tiles at a time
    static constexpr int NJ = NW / DS / KSP, LGROWS = NJ == 4 ? 7 : 6;   // 32 NJ = 2^LGROWS rows
    // LDS: K and V of a tile are TB bytes each
    static constexpr int TB = 32 * HD * ES;
    static constexpr int NK = DS == 2 ? 1 : 2 * KSP, NV = DS == 2 ? 1 : KSP == 2 ? 5 : 2;
    static constexpr int META = (NK + NV) * TB, XCH = META + 2 * KSP * 1024;
    static constexpr int RB = HD / DS * ES;                          // bytes of a wave's part of a row
    static constexpr int NEED = XCH + (DS == 2 ? NW * 4096 : 0);     // DS 2: partial scores
    static constexpr int ROWS = KSP == 1 ? NW * 32 * RB : 0;         // the output's rows
    static constexpr int LDS = NEED > ROWS ? NEED : ROWS;
    static constexpr int JOIN = NJ * (HD * 128 + 256);               // sums of waves 4 .. 7
    static_assert(LDS <= 160 * 1024 && NJ * DS * KSP == NW && (KSP == 1 || JOIN <= LDS), "LDS");
    static __device__ __forceinline__ int k_at(int st, int kp) { return DS == 2 ? 0 : ((st & 1) * KSP + kp) * TB; }
    static __device__ __forceinline__ int v_at(int st, int kp) {
        return (NK + (DS == 2 ? 0 : kp == 0 ? st & 1 : 2 + st % 3)) * TB;
    }
    static __device__ __forceinline__ int meta_at(int st, int kp) { return META + ((st & 1) * KSP + kp) * 1024; }
};

// of all 64 lanes, by lane moves within rows of 16 and four reads across them
template <typename Op>
__device__ __forceinline__ unsigned wave_reduce(unsigned v, Op op) {
    v = op(v, (unsigned)dpp_i<kDppXor1>((int)v));
    v = op(v, (unsigned)dpp_i<kDppXor2>((int)v));
    v = op(v, (unsigned)dpp_i<kDppHalfMirror>((int)v));
    v = op(v, (unsigned)dpp_i<kDppMirror>((int)v));
    auto at = [&](int l) { return (unsigned)__builtin_amdgcn_readlane((int)v, l); };
    return op(op(at(0), at(16)), op(at(32), at(48)));
}

// The u-th of all workgroups of a kv head, those with the most keys first: a
// sequence's c-th workgroup has the more keys the larger c is (up to the
// window), whatever sequence it is, so they go by c, downwards, and by
// sequence.  Up to 64 sequences, one a lane.  (In the order of the sequences a
// launch of one and a half rounds takes two: prompts of 100 to 2048 rows with
// a window of 512, fp32, 8 heads of 256: 120 -> 80 us.)
__device__ __forceinline__ bool longest_first(const PackedArgs& a, int nj, unsigned u, int& s, unsigned& c) {
    const int lane = threadIdx.x & 63;
    unsigned units = 0;
    if (lane < a.n_seqs) {
        const int r0 = a.cu[lane], r1 = a.cu[lane + 1];
        if (r0 >= 0 && r1 > r0 && r1 <= a.m) units = (unsigned)(((long)((r1 - r0 + 31) >> 5) * a.group + nj - 1) / nj);
    }
    // workgroups of all sequences from their c-th on
    auto from = [&](unsigned c) {
        return wave_reduce(units > c ? units - c : 0, [](unsigned x, unsigned y) { return x + y; });
    };
    if (u >= from(0)) return false;
    // the largest c with more than u from it on
    unsigned lo = 0, hi = wave_reduce(units, [](unsigned x, unsigned y) { return x > y ? x : y; });
    while (hi - lo > 1) {
        const unsigned mid = (lo + hi) >> 1;
        if (from(mid) > u) lo = mid;
        else hi = mid;
    }
    c = lo;
    unsigned long long have = __ballot(units > c);
    for (unsigned k = u - from(c + 1); k; k--) have &= have - 1;
    s = __builtin_ctzll(have);
    return true;
}

// a workgroup's sequence and jobs
struct Share {
    int r0, n;                  // the sequence's first row, its rows
    unsigned kvh, block0;       // its first block of K and V
    long job0, jobs, jl;        // the first job, the sequence's, the last of the workgroup
};
__device__ __forceinline__ bool find_share(const PackedArgs& a, int nj, int lg, Share& o) {
    const unsigned id = blockIdx.x, u = id / (unsigned)a.n_kv;
    o.kvh = id % (unsigned)a.n_kv;
    int s;
    unsigned c;
    if (a.n_seqs <= 64) {
        if (!longest_first(a, nj, u, s, c)) return false;
    } else {
        const unsigned back = gridDim.x / a.n_kv - 1 - u;   // a sequence's longest first
        s = unit_seq(a.cu, a.n_seqs, a.group, lg, a.extra, back);
        c = back - unit_base(a.cu, s, a.group, lg, a.extra);
    }
    const int r1 = a.cu[s + 1];
    o.r0 = a.cu[s];
    o.n = r1 - o.r0;
    if (o.r0 < 0 || r1 <= o.r0 || r1 > a.m) return false;
    o.block0 = unit_base(a.cu, s, 1, 5, 1);
    o.jobs = (long)((o.n + 31) >> 5) * a.group;
    o.job0 = (long)c * nj;
    if (o.job0 >= o.jobs) return false;
    o.jl = o.job0 + nj < o.jobs ? o.job0 + nj - 1 : o.jobs - 1;
    return true;
}

template <int T, int HD>
__global__ __launch_bounds__((64 * Plan<T, HD>::NW), (Plan<T, HD>::NW / 4)) void attn_packed_kernel(PackedArgs a) {
    typedef Plan<T, HD> P;
    typedef typename Kind<T>::t E;
    typedef typename Kind<T>::op op;
    constexpr int ES = P::ES, NS = Kind<T>::NS, NW = P::NW, DS = P::DS, NJ = P::NJ, KSP = P::KSP, TB = P::TB;
    constexpr int KS = HD / 16 / DS, NT = HD / 32 / DS;   // a wave's product steps and 32-dim tiles
    constexpr int kHalf = TB / 1024;                      // KB of a tile's K, of its V
    // how far a score may pass the maximum before it moves, and how far above the
    // largest score it is put.  bf16, whose V goes as far as fp32: weights are at
    // most 1; fp16's smallest numbers ask for large weights, and its V cannot overflow
    constexpr float kSlack = T == G4_F32 ? 4.0f : T == G4_F16 ? 8.0f : 0.0f, kRaise = T == G4_BF16 ? 8.0f : 0.0f;
    constexpr float kLift = T == G4_F32 ? 11.0f : 0.0f;   // fp16 weights: 2^11 above their fp32 size
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), part = wave % DS, kp = wave / (NJ * DS);

    Share sh;
    if (!find_share(a, NJ, P::LGROWS, sh)) return;
    const int r0 = sh.r0, n = sh.n;
    const long job0 = sh.job0, jobs = sh.jobs, jl = sh.jl;
    const unsigned kvh = sh.kvh;
    const int slot = wave / DS % NJ;
    const bool mine = job0 + slot < jobs;
    const long job = mine ? job0 + slot : jl;
    const int jt = (int)(job / a.group), head = (int)kvh * a.group + (int)(job - (long)jt * a.group);
    const int row = jt * 32 + col;                        // this lane's row of the sequence
    auto first_key = [&](int r) { return a.window > 0 && r >= a.window ? r + 1 - a.window : 0; };
    const int kt0 = first_key((int)(job0 / a.group) * 32) >> 5, kt1 = (int)(jl / a.group);
    // the stages that have a tile for this wave: s0 .. s1 - 1
    const int my0 = (first_key(jt * 32) >> 5) - kt0 - kp, my1 = jt - kt0 - kp;
    const int s0 = mine && my0 > 0 ? (my0 + KSP - 1) / KSP : 0, s1 = mine && my1 >= 0 ? my1 / KSP + 1 : s0;
    const int wfirst = first_key(row);
    // tiles that every row of the job sees whole lie between these
    const int full0 = (first_key(jt * 32 + 31) + 31) >> 5, full1 = jt - 1;

    // ---- tiles on their way into LDS: stage st has the tiles kt0 + KSP st + (0 .. KSP - 1) ----
    const int stages = (kt1 - kt0) / KSP + 1;
    const uint8_t* rec0 = a.work + ((size_t)(sh.block0 + kt0) * a.n_kv + kvh) * block_bytes(HD, ES);
    const size_t rec_step = (size_t)a.n_kv * block_bytes(HD, ES);
    constexpr int kShare = kHalf * KSP / NW;              // pieces a wave copies of a stage's K, of its V
    constexpr int kWhole = kHalf / NW;                    // of one tile's (0: half the waves have a tile each)
    static_assert(kHalf * KSP % NW == 0 && (kWhole || kShare == 1), "shares");
    const int first_piece = kWhole ? wave : wave % kHalf;
    // past the last tile: no bytes
    auto tile_rsrc = [&](int tile) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)(rec0 + tile * rec_step), 0,
                                                 tile <= kt1 - kt0 ? (int)block_bytes(HD, ES) : 0, kBufWord3);
    };
    auto stage = [&](int st, bool v) {
#pragma unroll
        for (int t = 0; t < (kWhole ? KSP : 1); t++) {
            const int tt = kWhole ? t : wave / kHalf;
            const __amdgpu_buffer_rsrc_t r = tile_rsrc(st * KSP + tt);
            uint8_t* at = lds + (v ? P::v_at(st, tt) : P::k_at(st, tt)) + first_piece * 1024;
#pragma unroll
            for (int i = 0; i < (kWhole ? kWhole : 1); i++)
                buf_load_lds16(r, at + i * NW * 1024, first_piece * 1024 + lane * 16, (v ? TB : 0) + i * NW * 1024);
            // the last half kilobyte (the other half: no such bytes)
            if (!v && (kWhole ? wave == t : first_piece == 0)) buf_load_lds16(r, lds + P::meta_at(st, tt), lane * 16, 2 * TB);
        }
    };
    auto stage_k = [&](int st) { stage(st, false); };
    auto stage_v = [&](int st) { stage(st, true); };
    stage_k(0);
    if (DS == 1) stage_v(0);

    // ---- q, through places in LDS that the first stage leaves free ----
    op q[NS][KS];
    float fq = fabsf(a.scale) * kLog2e;
    constexpr int kPasses = KSP == 2 ? 1 : 2, kChunks = P::RB / 16 / kPasses, kSteps = KS / kPasses;
    // fp32: half of the second K and V places each; 16 bits: the second K places
    // and free V ones, a job's rows by its two waves; DS 2: V and the partial scores
    uint8_t* box = lds + (KSP == 2 ? (slot < 2 ? 2 + slot : slot == 2 ? 5 : 7) * TB
                          : DS == 1 ? (wave < 2 ? TB : 2 * TB) + wave * (TB / 2)
                          : wave < 4 ? TB + wave * (TB / 4) : P::XCH + (wave - 4) * (TB / 4));
    auto q_row = [&](int pass) {
        return [=](int r) {
            const int i = jt * 32 + r < n ? jt * 32 + r : n - 1;
            return (const uint8_t*)((const E*)a.q + (size_t)(r0 + i) * a.q_stride + (size_t)head * HD + part * (HD / DS)) +
                   pass * kChunks * 16;
        };
    };
    auto chunk = [&](int c) { return box + row_slot<kChunks>(col, c); };
    if constexpr (T == G4_F32) {
        float4 x[KS][2];
        unsigned top = 0;
#pragma unroll
        for (int pass = 0; pass < 2; pass++) {
            rows_to_lds<kChunks, 32>(box, 0, q_row(pass));
#pragma unroll
            for (int i = 0; i < kSteps; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float4 y = *reinterpret_cast<const float4*>(chunk(i * 4 + h * 2 + j));
                    x[pass * kSteps + i][j] = y;
                    const float e[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const unsigned m = __float_as_uint(e[k]) & 0x7fffffffu;
                        top = m > top ? m : top;
                    }
                }
        }
        const unsigned o = __shfl_xor(top, 32, 64);
        top = o > top ? o : top;
        const int e = (int)(top >> 23) > kLowK ? (int)(top >> 23) : kLowK;
        float sf = row_scale(e < 255 ? e : 254);
        fq *= e < 255 ? row_scale_inv(e) : __uint_as_float(0x7fc00000u);
        if (a.scale < 0.0f) sf = -sf;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            h2v_t hi[4], lo[4];
            split2(x[i][0].x, x[i][0].y, sf, hi[0], lo[0]);
            split2(x[i][0].z, x[i][0].w, sf, hi[1], lo[1]);
            split2(x[i][1].x, x[i][1].y, sf, hi[2], lo[2]);
            split2(x[i][1].z, x[i][1].w, sf, hi[3], lo[3]);
            __builtin_memcpy(&q[0][i], hi, 16);
            __builtin_memcpy(&q[1][i], lo, 16);
        }
    } else {
        const unsigned flip = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
        for (int pass = 0; pass < kPasses; pass++) {
            if constexpr (KSP == 2) {
                rows_to_lds<kChunks, 16>(box, kp * 16, q_row(pass));
                lds_barrier();
            } else {
                rows_to_lds<kChunks, 32>(box, 0, q_row(pass));
            }
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
                uint4 x = *reinterpret_cast<const uint4*>(chunk(i * 2 + h));
                if (a.scale == 0.0f) x = make_uint4(0, 0, 0, 0);
                x.x ^= flip; x.y ^= flip; x.z ^= flip; x.w ^= flip;
                q[0][pass * kSteps + i] = __builtin_bit_cast(op, x);
            }
        }
        if (a.scale == 0.0f) fq = 1.0f;
    }
    // one wave a SIMD: q and o stay in the accumulation registers, from which
    // products take them as well (left to itself the compiler moves them there
    // and back for every tile)
    constexpr bool kAcc = T == G4_F32 && HD >= 256;
    if constexpr (kAcc) {
#pragma unroll
        for (int k = 0; k < NS; k++)
#pragma unroll
            for (int i = 0; i < KS; i++) {
                asm("" : "+a"(q[k][i]));
            }
    }
    f16_t o[NT] = {};
    float m = -FLT_MAX, l = 0.0f;
    f16_t sc;
    op p[NS][2];
    struct Ops {
        op x[NS];
    };
    // kFeed: the next tile's copies are issued between the products, one a step
    // (by themselves the 65 KB of an fp32 tile of 256 dims take the CU's address
    // unit 1000 of a tile's 6500 cycles, which nothing else would use), those
    // past the last tile as well: they have no bytes, and a branch costs more
    constexpr bool kFeed = NS == 2;
    auto scores = [&](int st) {
        const uint8_t* at = lds + P::k_at(st, kp) + lane * 16;
        sc = f16_t{};
        f16_t sx = {};
        if constexpr (kFeed) {
            const __amdgpu_buffer_rsrc_t r = tile_rsrc(st + 1);
            uint8_t* to[2] = {lds + P::k_at(st + 1, 0) + wave * 1024, lds + P::v_at(st + 1, 0) + wave * 1024};
            run_products<Ops, KS, 2>(
                [&](int i, Ops& k) {
#pragma unroll
                    for (int j = 0; j < NS; j++) k.x[j] = *reinterpret_cast<const op*>(at + j * 64 * HD + i * 1024);
                },
                [&](int i, const Ops& k) {
                    sc = mfma32(k.x[0], q[0][i], sc);
#pragma unroll
                    for (int j = i * 2 * kShare / KS; j < (i + 1) * 2 * kShare / KS; j++)
                        buf_load_lds16(r, to[j / kShare] + j % kShare * NW * 1024, wave * 1024 + lane * 16,
                                       j / kShare * TB + j % kShare * NW * 1024);
                    if (i == KS - 1 && wave == 0) buf_load_lds16(r, lds + P::meta_at(st + 1, 0), lane * 16, 2 * TB);
                    sx = mfma32(k.x[0], q[1][i], sx);
                    sx = mfma32(k.x[1], q[0][i], sx);
                });
            sc += sx;
        } else {
#pragma unroll
            for (int i = 0; i < KS; i++) sc = mfma32(*reinterpret_cast<const op*>(at + (part * KS + i) * 1024), q[0][i], sc);
            order_products<KS, 3, 1, 1>();
        }
    };
    auto weights = [&](int st, int kt) {
        const float* meta = reinterpret_cast<const float*>(lds + P::meta_at(st, kp));
        const unsigned* mk = reinterpret_cast<const unsigned*>(meta) + kMetaMask / 4;
        const unsigned marks = __builtin_amdgcn_readfirstlane(mk[0] | mk[1]);
        float vinv[16];
        if constexpr (T == G4_F32) {
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const float4 fk = *reinterpret_cast<const float4*>(meta + 8 * b + 4 * h);
                const float4 ve = *reinterpret_cast<const float4*>(meta + kMetaVExp / 4 + 8 * b + 4 * h);
                const float4 vi = *reinterpret_cast<const float4*>(meta + kMetaVInv / 4 + 8 * b + 4 * h);
                const float f[4] = {fk.x, fk.y, fk.z, fk.w}, e[4] = {ve.x, ve.y, ve.z, ve.w}, v[4] = {vi.x, vi.y, vi.z, vi.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sc[4 * b + i] = __builtin_fmaf(sc[4 * b + i], fq * f[i], e[i]);
                    vinv[4 * b + i] = v[i];
                }
            }
        }
        if (marks) {
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (marks >> (8 * (r >> 2) + 4 * h + (r & 3)) & 1) sc[r] = __uint_as_float(0x7fc00000u);
        }
        if (kt < full0 || kt > full1) {
            const int hi = row - kt * 32 - 4 * h, lo = wfirst - kt * 32 - 4 * h;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int key = 8 * (r >> 2) + (r & 3);
                if (key > hi || key < lo) sc[r] = -INFINITY;
            }
        }
        float top = sc[0];
#pragma unroll
        for (int r = 1; r < 16; r++) top = fmaxf(top, sc[r]);
        if constexpr (T != G4_F32) top *= fq;
        if (__any(top > m + kSlack)) {
            top = fmaxf(top, shfl_xor(top, 32));
            top = fmaxf(top + kRaise, m);
            const float f = exp2f(m - top);
            if constexpr (T == G4_F32) l = move_sum(l, m - top);
            else l *= f;
            m = top;
#pragma unroll
            for (int i = 0; i < NT; i++) o[i] *= f;
        }
        const float base = m - kLift;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = sc[8 * t + j];
                w[j] = __builtin_amdgcn_exp2f(T == G4_F32 ? x - base : __builtin_fmaf(x, fq, -base));
                if constexpr (T == G4_F32) l = __builtin_fmaf(w[j], vinv[8 * t + j], l);
                else l += w[j];
            }
            if constexpr (T == G4_F32) {
                h2v_t hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 4; j++) split2(w[2 * j], w[2 * j + 1], 1.0f, hi[j], lo[j]);
                __builtin_memcpy(&p[0][t], hi, 16);
                __builtin_memcpy(&p[1][t], lo, 16);
            } else {
                // Rounded to the type, the operand's, while l keeps fp32: bf16, 8191 rows, 8
                // heads of 256, 283 us with an error of 0.00205 of the norm, where the
                // output's own rounding alone makes 0.00166.  That is reached by two
                // products, of hi and lo, in 399 us, or by fp16 weights and V rows with
                // exponents as in fp32 in 328 (more instructions a key, the SIMD's
                // registers spent); of 512, four prompts of 4096: 622 (0.00211), 828, 684.
#pragma unroll
                for (int j = 0; j < 8; j++) p[0][t][j] = (E)w[j];
            }
        }
        if constexpr (T == G4_F32) {
            const float lost = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(meta[kMetaLost / 4])));
            if (__any(l < lost)) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = 8 * (r >> 2) + 4 * h + (r & 3);
                    l += lost_weight(sc[r] - base, meta[kMetaVExp / 4 + key], vinv[r]);
                }
            }
        }
    };
    auto values = [&](int st) {
        const uint8_t* at = lds + P::v_at(st, kp) + lane * 16;
        if constexpr (NS == 2) {
            run_products<Ops, 2 * NT, 2>(
                [&](int i, Ops& v) {
#pragma unroll
                    for (int j = 0; j < NS; j++) v.x[j] = *reinterpret_cast<const op*>(at + j * 64 * HD + i * 1024);
                },
                [&](int i, const Ops& v) {
                    f16_t& s = o[i >> 1];
                    s = mfma32(v.x[0], p[0][i & 1], s);
                    s = mfma32(v.x[0], p[1][i & 1], s);
                    s = mfma32(v.x[1], p[0][i & 1], s);
                });
        } else {
#pragma unroll
            for (int i = 0; i < 2 * NT; i++)
                o[i >> 1] = mfma32(*reinterpret_cast<const op*>(at + (part * NT * 2 + i) * 1024), p[0][i & 1], o[i >> 1]);
            order_products<2 * NT, 3, 1, 1>();
        }
    };

    if constexpr (DS == 1) {
        // this wave's copies have landed, then everyone's; and all are done
        // with the stage before (waves 4 .. 7 but for its V, which has three
        // places)
        auto turn = [&](int st, bool feed) {
            wait_vm<0>();
            lds_barrier();
            if (!feed && st + 1 < stages) {
                stage_k(st + 1);
                stage_v(st + 1);
            }
        };
        int st = 0;
        for (; st < s0; st++) turn(st, false);
        if (KSP == 1 || kp == 0) {
            for (; st < s1; st++) {
                turn(st, kFeed);
                scores(st);
                weights(st, kt0 + st * KSP + kp);
                values(st);
            }
        } else if (s0 < s1) {
            turn(st, false);
            scores(st);
            weights(st, kt0 + st * KSP + kp);
            for (st++; st < s1; st++) {
                turn(st, false);
                values(st - 1);
                scores(st);
                weights(st, kt0 + st * KSP + kp);
            }
            if (st < stages) turn(st, false);
            values(s1 - 1);
            st++;
        }
        for (; st < stages; st++) turn(st, false);
    } else {
        // a tile's turn up to its scores, and from there on; both waves of a job
        // take part in the same ones
        f4_t* box = reinterpret_cast<f4_t*>(lds + P::XCH);
        auto begin = [&](int st) {
            wait_vm<0>();
            lds_barrier();   // K is there, V of the tile before done with
            stage_v(st);
        };
        auto middle = [&](int st) {
            lds_barrier();   // K is done with, the partial scores there
            if (st + 1 < stages) stage_k(st + 1);
        };
        auto end = [&](int st) {
            // all copies but those of the next K (and, wave 0, its factors)
            if (st + 1 >= stages) wait_vm<0>();
            else if (wave == 0) wait_vm<kShare + 1>();
            else wait_vm<kShare>();
            lds_barrier();   // V is there
        };
        int st = 0;
        for (; st < s0; st++) {
            begin(st);
            middle(st);
            end(st);
        }
        for (; st < s1; st++) {
            begin(st);
            scores(st);
#pragma unroll
            for (int i = 0; i < 4; i++)
                box[(wave * 4 + i) * 64 + lane] = f4_t{sc[4 * i], sc[4 * i + 1], sc[4 * i + 2], sc[4 * i + 3]};
            middle(st);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f4_t y = box[((wave ^ 1) * 4 + i) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; j++) sc[4 * i + j] += y[j];
            }
            weights(st, kt0 + st);
            end(st);
            values(st);
        }
        for (; st < stages; st++) {
            begin(st);
            middle(st);
            end(st);
        }
    }

    if constexpr (KSP == 2) {
        // waves 4 .. 7 hand their sums to waves 0 .. 3
        wait_vm<0>();
        lds_barrier();
        float* ml = reinterpret_cast<float*>(lds + NJ * HD * 128) + slot * 64 + col * 2;
        f4_t* box = reinterpret_cast<f4_t*>(lds) + slot * HD * 8 + lane;
        l += shfl_xor(l, 32);
        if (kp == 1) {
            if (h == 0) {
                ml[0] = m;
                ml[1] = l;
            }
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int b = 0; b < 4; b++)
                    box[(i * 4 + b) * 64] = f4_t{o[i][4 * b], o[i][4 * b + 1], o[i][4 * b + 2], o[i][4 * b + 3]};
        }
        lds_barrier();
        if (kp == 1) return;
        const float m1 = ml[0], l1 = ml[1], top = fmaxf(m, m1);
        const float f0 = exp2f(m - top), f1 = exp2f(m1 - top);
        l = l * f0 + l1 * f1;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const f4_t y = box[(i * 4 + b) * 64];
#pragma unroll
                for (int j = 0; j < 4; j++) o[i][4 * b + j] = o[i][4 * b + j] * f0 + y[j] * f1;
            }
    } else {
        l += shfl_xor(l, 32);
    }
    // ---- the output's rows, where K and V (16 bits: this wave's other sums) were ----
    if (KSP == 1) {
        wait_vm<0>();
        lds_barrier();
    }
    if (!mine) return;
    wave_lds_order();
    const float f = 1.0f / l;
    constexpr int kRow = P::RB / 16;
    uint8_t* rows = lds + (KSP == 2 ? slot * HD * 128 : wave * 32 * P::RB);
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            E y[4];
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = (E)(o[i][4 * b + j] * f);
            uint8_t* to = rows + (ES == 4 ? row_slot<kRow>(col, i * 8 + 2 * b + h) : row_slot<kRow>(col, i * 4 + b) + h * 8);
            __builtin_memcpy(__builtin_assume_aligned(to, 4 * ES), y, 4 * ES);
        }
    rows_from_lds<kRow>(rows, n - jt * 32, [&](int r) {
        return (uint8_t*)((E*)a.out + (size_t)(r0 + jt * 32 + r) * a.out_stride + (size_t)head * HD + part * (HD / DS));
    });
}

// ---- fp32 at head_dim 512 ------------------------------------------------------------
// q and o of a job's 512 dims take two waves' registers.  Each wave computes
// the scores of 16 of a tile's 32 keys over all dims (q whole: the 256
// accumulation registers) and their weights, and adds all 32 keys' values to
// half the dims; the weights meet in LDS, with the maxima they stand for.  The
// maxima are whole numbers, so that weights of one are brought to another's by
// an exact power of two, which after the first tiles is 1.  Against halving
// the dims of both products (partial scores of all keys in LDS, weights
// computed twice, one barrier more): 2441 -> 1886 us over four prompts of 4096
// with the reads ahead, 1780 with q and the output as whole lines, 1640 with the
// copies between the products, 335 TFLOP/s.
// Bound by its copies to LDS, 128 KB a tile and 64 rows at 55 bytes/ns a CU
// (half of the time by themselves), and by the products; more rows do not fit
// the registers.
// K and V of a tile have one place each: the next K is on its way during the
// second product, V during the first.
struct Wide {
    static constexpr int HD = 512, TB = 32 * HD * 4, NJ = 2;
    static constexpr int META = 2 * TB, PW = META + 2048, MX = PW + NJ * 4096, LDS = MX + NJ * 2 * 32 * 8;
};
__global__ __launch_bounds__(256, 1) void attn_packed_wide_kernel(PackedArgs a) {
    constexpr int HD = Wide::HD, TB = Wide::TB, NJ = Wide::NJ, KS = HD / 32, NT = HD / 64;
    constexpr float kSlack = 4.0f, kLift = 11.0f;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, h = lane >> 5, c16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), part = wave & 1, slot = wave >> 1;
    Share sh;
    if (!find_share(a, NJ, 6, sh)) return;
    const bool mine = sh.job0 + slot < sh.jobs;
    const long job = mine ? sh.job0 + slot : sh.jl;
    const int jt = (int)(job / a.group), head = (int)sh.kvh * a.group + (int)(job - (long)jt * a.group);
    auto first_key = [&](int r) { return a.window > 0 && r >= a.window ? r + 1 - a.window : 0; };
    const int kt0 = first_key((int)(sh.job0 / a.group) * 32) >> 5, kt1 = (int)(sh.jl / a.group);
    const int my0 = (first_key(jt * 32) >> 5) - kt0, my1 = jt - kt0;
    const int s0 = mine && my0 > 0 ? my0 : 0, s1 = mine && my1 >= 0 ? my1 + 1 : s0;
    const int full0 = (first_key(jt * 32 + 31) + 31) >> 5, full1 = jt - 1;
    const int stages = kt1 - kt0 + 1;
    const uint8_t* rec0 = a.work + ((size_t)(sh.block0 + kt0) * a.n_kv + sh.kvh) * block_bytes(HD, 4);
    const size_t rec_step = (size_t)a.n_kv * block_bytes(HD, 4);
    // past the last tile: no bytes
    auto tile_rsrc = [&](int st) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)(rec0 + st * rec_step), 0, st < stages ? (int)block_bytes(HD, 4) : 0,
                                                 kBufWord3);
    };
    // a wave's of a tile's K, of its V, issued between its first kFeed steps of
    // products (all before the products 1780 us, over 4, 8, 16 steps 1695, 1640, 1652)
    constexpr int kCopies = TB / 4096, kFeed = 8;
    auto copy = [&](const __amdgpu_buffer_rsrc_t r, int st, bool v, int i) {
        buf_load_lds16(r, lds + (v ? TB : 0) + wave * 1024 + i * 4096, wave * 1024 + lane * 16, (v ? TB : 0) + i * 4096);
        if (!v && i == 0 && wave == 0) buf_load_lds16(r, lds + Wide::META + (st & 1) * 1024, lane * 16, 2 * TB);
    };
    auto stage = [&](int st, bool v) {
        const __amdgpu_buffer_rsrc_t r = tile_rsrc(st);
#pragma unroll
        for (int i = 0; i < kCopies; i++) copy(r, st, v, i);
    };
    // ---- q: rows c16 and 16 + c16, steps of 32 dims, 8 of them a lane; half of
    // the job's rows by each of its waves through LDS ----
    uint8_t* box = lds + slot * 32 * HD * 4;
    rows_to_lds<HD / 4, 16>(box, part * 16, [&](int r) {
        const int i = jt * 32 + r < sh.n ? jt * 32 + r : sh.n - 1;
        return (const uint8_t*)((const float*)a.q + (size_t)(sh.r0 + i) * a.q_stride + (size_t)head * HD);
    });
    lds_barrier();
    h8_t q[2][2][KS];
    float fq[2];
    int row2[2], wf2[2];
#pragma unroll
    for (int ct = 0; ct < 2; ct++) {
        row2[ct] = jt * 32 + 16 * ct + c16;
        wf2[ct] = first_key(row2[ct]);
        float4 x[KS][2];
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                x[i][j] = *reinterpret_cast<const float4*>(box + row_slot<HD / 4>(16 * ct + c16, i * 8 + g * 2 + j));
                const float e[4] = {x[i][j].x, x[i][j].y, x[i][j].z, x[i][j].w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const unsigned b = __float_as_uint(e[k]) & 0x7fffffffu;
                    top = b > top ? b : top;
                }
            }
#pragma unroll
        for (int d = 16; d < 64; d <<= 1) {
            const unsigned o = __shfl_xor(top, d, 64);
            top = o > top ? o : top;
        }
        const int e = (int)(top >> 23) > kLowK ? (int)(top >> 23) : kLowK;
        float sf = row_scale(e < 255 ? e : 254);
        fq[ct] = fabsf(a.scale) * kLog2e * (e < 255 ? row_scale_inv(e) : __uint_as_float(0x7fc00000u));
        if (a.scale < 0.0f) sf = -sf;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            h2v_t hi[4], lo[4];
            split2(x[i][0].x, x[i][0].y, sf, hi[0], lo[0]);
            split2(x[i][0].z, x[i][0].w, sf, hi[1], lo[1]);
            split2(x[i][1].x, x[i][1].y, sf, hi[2], lo[2]);
            split2(x[i][1].z, x[i][1].w, sf, hi[3], lo[3]);
            __builtin_memcpy(&q[0][ct][i], hi, 16);
            __builtin_memcpy(&q[1][ct][i], lo, 16);
            asm("" : "+a"(q[0][ct][i]));
            asm("" : "+a"(q[1][ct][i]));
        }
    }

    lds_barrier();   // q has been read
    stage(0, false);
    f16_t o[NT] = {};
    float m[2] = {-FLT_MAX, -FLT_MAX}, l[2] = {}, mo = -FLT_MAX;   // of rows row2, and of row col: what o stands for
    // the job's weights: [step of 16 keys][hi, lo][lane] 16 bytes; maxima: [part][row]
    struct Ops {
        h8_t x[2];
    };
    uint8_t* pw = lds + Wide::PW + slot * 4096;
    float* mx = reinterpret_cast<float*>(lds + Wide::MX) + slot * 64;
    auto scores = [&](int st) {
        const int kt = kt0 + st;
        const uint8_t* at = lds + (g >> 1) * 1024 + ((g & 1) * 32 + 16 * part + c16) * 16;
        f4_t sc[2] = {}, sx[2] = {};
        const __amdgpu_buffer_rsrc_t r = tile_rsrc(st);
        run_products<Ops, KS, 3>(
            [&](int i, Ops& k) {
                k.x[0] = *reinterpret_cast<const h8_t*>(at + i * 2048);
                k.x[1] = *reinterpret_cast<const h8_t*>(at + 64 * HD + i * 2048);
            },
            [&](int i, const Ops& k) {
#pragma unroll
                for (int ct = 0; ct < 2; ct++) sc[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.x[0], q[0][ct][i], sc[ct], 0, 0, 0);
                if (i < kFeed)
#pragma unroll
                    for (int j = i * kCopies / kFeed; j < (i + 1) * kCopies / kFeed; j++) copy(r, st, true, j);
#pragma unroll
                for (int ct = 0; ct < 2; ct++) sx[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.x[0], q[1][ct][i], sx[ct], 0, 0, 0);
#pragma unroll
                for (int ct = 0; ct < 2; ct++) sx[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.x[1], q[0][ct][i], sx[ct], 0, 0, 0);
            });
        // ---- weights of keys 16 part + 4 g .. + 3 ----
        const float* meta = reinterpret_cast<const float*>(lds + Wide::META + (st & 1) * 1024);
        const int key0 = 16 * part + 4 * g;
        const unsigned* mk = reinterpret_cast<const unsigned*>(meta) + kMetaMask / 4;
        const unsigned marks = __builtin_amdgcn_readfirstlane(mk[0] | mk[1]);
        const float4 fk = *reinterpret_cast<const float4*>(meta + key0), ve = *reinterpret_cast<const float4*>(meta + kMetaVExp / 4 + key0),
                     vi = *reinterpret_cast<const float4*>(meta + kMetaVInv / 4 + key0);
        const float f[4] = {fk.x, fk.y, fk.z, fk.w}, e[4] = {ve.x, ve.y, ve.z, ve.w}, v[4] = {vi.x, vi.y, vi.z, vi.w};
        float y[2][4], top[2];
#pragma unroll
        for (int ct = 0; ct < 2; ct++) {
#pragma unroll
            for (int r = 0; r < 4; r++) y[ct][r] = __builtin_fmaf(sc[ct][r] + sx[ct][r], fq[ct] * f[r], e[r]);
            if (marks) {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (marks >> (key0 + r) & 1) y[ct][r] = __uint_as_float(0x7fc00000u);
            }
            if (kt < full0 || kt > full1) {
                const int hi = row2[ct] - kt * 32 - key0, lo = wf2[ct] - kt * 32 - key0;
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (r > hi || r < lo) y[ct][r] = -INFINITY;
            }
            top[ct] = fmaxf(fmaxf(y[ct][0], y[ct][1]), fmaxf(y[ct][2], y[ct][3]));
        }
        if (__any(top[0] > m[0] + kSlack || top[1] > m[1] + kSlack)) {
#pragma unroll
            for (int ct = 0; ct < 2; ct++) {
                float t = fmaxf(top[ct], shfl_xor(top[ct], 16));
                t = fmaxf(ceilf(fmaxf(t, shfl_xor(t, 32))), m[ct]);
                l[ct] = move_sum(l[ct], m[ct] - t);
                m[ct] = t;
            }
        }
        const float lost = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(meta[kMetaLost / 4])));
#pragma unroll
        for (int ct = 0; ct < 2; ct++) {
            const float base = m[ct] - kLift;
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                w[r] = __builtin_amdgcn_exp2f(y[ct][r] - base);
                l[ct] = __builtin_fmaf(w[r], v[r], l[ct]);
            }
            h2v_t hi[2], lo[2];
            split2(w[0], w[1], 1.0f, hi[0], lo[0]);
            split2(w[2], w[3], 1.0f, hi[1], lo[1]);
            // lane 32 h + row of step `part` takes keys 4 h .. + 3 and 8 + 4 h .. + 3 of the 16
            uint8_t* to = pw + part * 2048 + ((g & 1) * 32 + 16 * ct + c16) * 16 + (g >> 1) * 8;
            *reinterpret_cast<uint2*>(to) = make_uint2(h2_bits(hi[0]), h2_bits(hi[1]));
            *reinterpret_cast<uint2*>(to + 1024) = make_uint2(h2_bits(lo[0]), h2_bits(lo[1]));
            if (g == 0) mx[part * 32 + 16 * ct + c16] = m[ct];
        }
        if (__any(fminf(l[0], l[1]) < lost)) {
#pragma unroll
            for (int ct = 0; ct < 2; ct++)
#pragma unroll
                for (int r = 0; r < 4; r++) l[ct] += lost_weight(y[ct][r] - (m[ct] - kLift), e[r], v[r]);
        }
    };
    auto values = [&](int next) {
        const __amdgpu_buffer_rsrc_t r = tile_rsrc(next);
        h8_t p[2][2];   // [hi, lo][step]
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int k = 0; k < 2; k++) p[k][t] = *reinterpret_cast<const h8_t*>(pw + t * 2048 + k * 1024 + lane * 16);
        const float ma = mx[col], mb = mx[32 + col], top = fmaxf(ma, mb);
        if (__any(ma != mb || top != mo)) {
            const float fo = exp2f(mo - top);
            mo = top;
            // by 2^-24 at most at a time, fp16's smallest number
            auto scale = [&](float d, int t) {
                const _Float16 f0 = (_Float16)exp2f(fmaxf(d, -24.0f)), f1 = (_Float16)exp2f(fminf(d + 24.0f, 0.0f));
#pragma unroll
                for (int k = 0; k < 2; k++) p[k][t] = p[k][t] * f0 * f1;
            };
            scale(ma - top, 0);
            scale(mb - top, 1);
#pragma unroll
            for (int i = 0; i < NT; i++) o[i] *= fo;
#pragma unroll
            for (int ct = 0; ct < 2; ct++) {
                const float t = fmaxf(mx[16 * ct + c16], mx[32 + 16 * ct + c16]);
                l[ct] = move_sum(l[ct], m[ct] - t);
                m[ct] = t;
            }
        }
        const uint8_t* at = lds + TB + part * NT * 2048 + lane * 16;
        run_products<Ops, 2 * NT, 2>(
            [&](int i, Ops& v) {
                v.x[0] = *reinterpret_cast<const h8_t*>(at + i * 1024);
                v.x[1] = *reinterpret_cast<const h8_t*>(at + 64 * HD + i * 1024);
            },
            [&](int i, const Ops& v) {
                f16_t& s = o[i >> 1];
                s = mfma32(v.x[0], p[0][i & 1], s);
                if (i < kFeed)
#pragma unroll
                    for (int j = i * kCopies / kFeed; j < (i + 1) * kCopies / kFeed; j++) copy(r, next, false, j);
                s = mfma32(v.x[0], p[1][i & 1], s);
                s = mfma32(v.x[1], p[0][i & 1], s);
            });
    };

    auto begin = [&]() {
        wait_vm<0>();
        lds_barrier();   // K is there, V and the weights of the tile before are done with
    };
    auto middle = [&]() {
        wait_vm<0>();
        lds_barrier();   // V and the weights are there, K is done with
    };
    auto pass = [&](int st) {
        begin();
        stage(st, true);
        middle();
        stage(st + 1, false);
    };
    int st = 0;
    for (; st < s0; st++) pass(st);
    for (; st < s1; st++) {
        begin();
        scores(st);
        middle();
        values(st + 1);
    }
    for (; st < stages; st++) pass(st);

    // ---- the two waves' weight sums ----
    float* ls = reinterpret_cast<float*>(lds + Wide::MX) + 128 + slot * 64;
#pragma unroll
    for (int ct = 0; ct < 2; ct++) {
        l[ct] += shfl_xor(l[ct], 16);
        l[ct] += shfl_xor(l[ct], 32);
        if (g == 0) ls[part * 32 + 16 * ct + c16] = l[ct];
    }
    wait_vm<0>();
    lds_barrier();
    if (!mine) return;
    const float f = 1.0f / (ls[col] + ls[32 + col]);
    uint8_t* rows = lds + wave * 32 * HD * 2;
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int b = 0; b < 4; b++)
            *reinterpret_cast<f4_t*>(rows + row_slot<HD / 8>(col, i * 8 + 2 * b + h)) =
                f4_t{o[i][4 * b] * f, o[i][4 * b + 1] * f, o[i][4 * b + 2] * f, o[i][4 * b + 3] * f};
    rows_from_lds<HD / 8>(rows, sh.n - jt * 32, [&](int r) {
        return (uint8_t*)((float*)a.out + (size_t)(sh.r0 + jt * 32 + r) * a.out_stride + (size_t)head * HD + part * (HD / 2));
    });
}

template <int T, int HD>
int launch_packed(PackedArgs a) {
    typedef Plan<T, HD> P;
    const double keys = a.window > 0 && a.window < a.m ? a.window : a.m;
    if ((double)a.m * keys * a.n_heads <= kFewPairs) {
        hipLaunchKernelGGL((attn_packed_few_kernel<T, HD>), dim3(a.m, a.n_heads), dim3(256), 0, g4_stream(), a);
        return g4_check_launch("attn_packed_few_kernel");
    }
    // a sequence of n rows has ceil(ceil(n / 32) group / NJ) units, at most
    // n group / (32 NJ) + extra
    a.extra = (31 * a.group + 32 * (P::NJ - 1) + 32 * P::NJ - 1) / (32 * P::NJ);
    const size_t units = (((size_t)a.m * a.group) >> P::LGROWS) + (size_t)a.extra * a.n_seqs;
    constexpr bool kWide = T == G4_F32 && HD == 512;
    constexpr int kLds = kWide ? Wide::LDS : P::LDS, kThreads = 64 * P::NW;
    G4_CHECK_ARG(kv_grid_fits(units * a.n_kv, kThreads) && kv_grid_fits((size_t)a.m / 32 + a.n_seqs, 256),
                 "g4_attn_prompt_packed: %d rows of %d sequences, %d heads: more than one launch takes", a.m, a.n_seqs,
                 a.n_heads);
    void (*kernel)(PackedArgs);
    if constexpr (kWide) kernel = attn_packed_wide_kernel;
    else kernel = attn_packed_kernel<T, HD>;
    // more than 64 KB of LDS has to be asked for, once on each device
    static std::atomic<unsigned long long> asked{0};
    int dev = 0;
    G4_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !(asked >> dev & 1)) {
        G4_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
        if (dev < 64) asked |= 1ull << dev;
    }
    hipLaunchKernelGGL((packed_layout_kernel<T, HD>), dim3(a.m / 32 + a.n_seqs, a.n_kv, 2), dim3(256), 0, g4_stream(), a);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(units * a.n_kv)), dim3(kThreads), kLds, g4_stream(), a);
    return g4_check_launch("attn_packed_kernel");
}
template <int T>
int launch_packed(const PackedArgs& a, int hd) {
    if (hd == 64) return launch_packed<T, 64>(a);
    if (hd == 128) return launch_packed<T, 128>(a);
    if (hd == 256) return launch_packed<T, 256>(a);
    return launch_packed<T, 512>(a);
}

int packed_size(int type) { return type == G4_F32 ? 4 : type == G4_F16 || type == G4_BF16 ? 2 : 0; }

}  // namespace
}  // namespace g4

using namespace g4;

extern "C" size_t g4_attn_prompt_packed_work_bytes(int type, int n_seqs, int m, int n_kv, int hd) {
    if (!packed_size(type) || n_seqs < 1 || n_seqs > kKvMaxSeqs || m < 1 || n_kv < 1 || n_kv > 65535 ||
        (hd != 64 && hd != 128 && hd != 256 && hd != 512))
        return 0;
    return ((size_t)m / 32 + n_seqs) * n_kv * block_bytes(hd, packed_size(type));
}

extern "C" int g4_attn_prompt_packed(const void* q, int q_stride, const void* k, const void* v, int kv_stride, void* out,
                                     int out_stride, int type, const int* cu, int n_seqs, int m, int window, int n_heads,
                                     int n_kv, int hd, float attn_scale, void* work) {
    const char* who = "g4_attn_prompt_packed";
    G4_CHECK(packed_size(type), G4_ERR_TYPE, "%s: unsupported type %d", who, type);
    G4_CHECK_ARG(g4_attn_prompt_packed_work_bytes(type, n_seqs, m, n_kv, hd),
                 "%s: bad sizes (%d rows of %d sequences (1 to %d), %d kv heads of %d)", who, m, n_seqs, kKvMaxSeqs, n_kv,
                 hd);
    G4_CHECK_ARG(n_heads > 0 && n_heads <= 65535 && n_heads % n_kv == 0 && window >= 0,
                 "%s: %d heads over %d kv heads, window %d", who, n_heads, n_kv, window);
    G4_CHECK_ARG(q && k && v && out && cu && work && al16(q) && al16(k) && al16(v) && al16(out) && al16(work),
                 "%s: null or unaligned pointer", who);
    const int unit = 16 / packed_size(type);
    G4_CHECK_ARG(q_stride % unit == 0 && kv_stride % unit == 0 && out_stride % unit == 0 && q_stride / hd >= n_heads &&
                 kv_stride / hd >= n_kv && out_stride / hd >= n_heads,
                 "%s: strides %d, %d, %d (multiples of %d, heads * hd at least)", who, q_stride, kv_stride, out_stride, unit);
    PackedArgs a = {};
    a.q = q; a.k = k; a.v = v; a.out = out; a.work = (uint8_t*)work; a.cu = cu; a.q_stride = q_stride;
    a.kv_stride = kv_stride; a.out_stride = out_stride; a.n_seqs = n_seqs; a.m = m; a.window = window;
    a.n_heads = n_heads; a.n_kv = n_kv; a.group = n_heads / n_kv; a.scale = attn_scale;
    if (type == G4_F32) return launch_packed<G4_F32>(a, hd);
    if (type == G4_F16) return launch_packed<G4_F16>(a, hd);
    return launch_packed<G4_BF16>(a, hd);
}
