// attn_chunk.hip -- attention of chunks of new rows of every sequence over the
// paged KV cache, which holds their own keys and values already.
#include <atomic>

#include "g4_attn_tile.h"
#include "g4_kvpage.h"

namespace g4 {
namespace {

constexpr int kLgShares = 8, kShares = 1 << kLgShares;   // workgroups that share the work, one a CU
// Keys that stand for what it costs to begin and to end an item.  us with 32, 64, 96,
// 160, 224 and 320 (8 q heads on 2 kv heads): 40 sequences of a row and one of 471, bf16
// of 512: 93, 92, 84, 81, 80, 84; nine of 3416 rows, fp32 of 256 under a window of 512:
// 106, 97, 96, 94, 104, 105; 32 of 4 to 8 rows, fp32 over codes of 512: 66, 59, 59, 59, 61, 60:
// anything from 96 to 224 would do.
constexpr int kLead = 160;
// No smaller share than this.  Against 96: 204 rows of 4 sequences, fp32 of 256, 29 us
// against 35, 571 rows of 31, bf16 of 512, 23 against 36 (one call 21 against 19).
constexpr int kLeast = 48;
constexpr double kFewKeys = 256, kFewPairs = 1 << 17;

struct ChunkArgs {
    KvPool p;
    const void* q;
    void* out;
    const int* cu;
    const int* lens;
    float* part;
    int q_stride, out_stride, n_seqs, m, window, n_heads;
    int group;      // q heads a kv head
    int gh, ngrp;   // of these, a workgroup's; groups of them
    int rpi;        // rows of an item
    int lg;         // no more shares than 2^lg, by the call's sizes
    bool pairs;     // Mode::kPairs
    int cols;       // columns of a partial result, a multiple of 32
    float scale;
    float fq, by;   // rows of 16 bits: what a sum of products is multiplied by; SMALL: the rows before
};

// ---- shares of the work ------------------------------------------------------
// An item is up to rpi rows of a sequence, a kv head and up to gh of its q
// heads: at most a workgroup's columns.  Its measure is the keys it looks at
// (rpi rows counted whole) and kLead.  All items form one line, by sequence,
// kv head, group of heads and row, and share w of W takes the measure N w / W
// .. N (w + 1) / W - 1 of it, whatever the lengths are: a few rows of a long
// sequence are spread over many workgroups, short sequences share one.  The
// line's sums over a sequence's items are closed forms.

typedef unsigned long long u64;

struct Seq {
    int r0, n, hist;   // first row, rows (0: none, or what does not fit), earlier positions
};
__device__ __forceinline__ Seq seq_of(const ChunkArgs& a, int r0, int r1, int len) {
    Seq q = {r0, r1 - r0, len - (r1 - r0)};
    if (r0 < 0 || r1 <= r0 || r1 > a.m || q.n > len || !a.p.fits(len)) q.n = 0;
    return q;
}
__device__ __forceinline__ int seq_items(const ChunkArgs& a, const Seq& q) {
    return (int)(((unsigned)q.n + a.rpi - 1) / (unsigned)a.rpi);
}
__device__ __forceinline__ int first_key(const ChunkArgs& a, int pos) {
    return a.window > 0 && pos >= a.window ? pos + 1 - a.window : 0;
}
// measure of item i, and of the first c items: hist + (i + 1) rpi keys while
// the window does not pass the first of them, window - 1 + rpi from there on
__device__ __forceinline__ u64 item_measure(const ChunkArgs& a, const Seq& q, int i) {
    const u64 row = (u64)i * a.rpi;
    if (a.window > 0 && q.hist + row >= (u64)a.window) return (u64)kLead + a.window - 1 + a.rpi;
    return kLead + q.hist + row + a.rpi;
}
__device__ __forceinline__ u64 items_measure(const ChunkArgs& a, const Seq& q, int c) {
    u64 whole = c;
    if (a.window > 0) {
        whole = q.hist < a.window ? (u64)((unsigned)(a.window - 1 - q.hist) / (unsigned)a.rpi) + 1 : 0;
        if (whole > (u64)c) whole = c;
    }
    return (u64)c * kLead + whole * q.hist + (u64)a.rpi * (whole * (whole + 1) / 2) +
           (c - whole) * ((u64)a.rpi + a.window - 1);
}

// a place on the line
struct Place {
    int s, rep, item;   // sequence, kv head and group of heads, item
    Seq q;
    u64 x, size;        // where in the item, the item's measure
};
struct Line {
    u64 total;
    int lg;             // W = 2^lg
    // where share w begins: N w / W without overflow
    __device__ __forceinline__ u64 at(unsigned w) const {
        return (total >> lg) * w + (((unsigned)total & ((1u << lg) - 1)) * w >> lg);
    }
};
__device__ __forceinline__ Line line_of(const ChunkArgs& a, u64 total) {
    const u64 most = total / kLeast;
    const int lg = 63 - __builtin_clzll(most | 1);
    return {total, lg < a.lg ? lg : a.lg};
}

constexpr u64 kNowhere = ~(u64)0;
// inclusive prefix sums over a wave: within rows of 16 by lane moves (lane -
// 1, 2, 4, 8, nothing from before the row), then the totals of the rows before
template <int CTRL>
__device__ __forceinline__ u64 row_shr(u64 v) {
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, 0xf, 0xf, true);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, 0xf, 0xf, true);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 lane_u64(u64 v, int l) {
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (unsigned)__builtin_amdgcn_readlane((int)v, l);
}
__device__ __forceinline__ u64 wave_scan(u64 v) {
    v += row_shr<0x111>(v);
    v += row_shr<0x112>(v);
    v += row_shr<0x114>(v);
    v += row_shr<0x118>(v);
    const u64 a = lane_u64(v, 15), b = a + lane_u64(v, 31), c = b + lane_u64(v, 47);
    const unsigned row = (threadIdx.x & 63) >> 4;
    return v + (row == 0 ? 0 : row == 1 ? a : row == 2 ? b : c);
}

// The line, and the place at(line) on it, by all NT threads of a workgroup
// (red: NT / 64 + 3 words of LDS): up to 64 sequences each wave by itself,
// after one round trip to memory.  false: no such place.
template <int NT, typename At>
__device__ __forceinline__ bool find_place(const ChunkArgs& a, At at, Line& line, Place& o, u64* red) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const unsigned rep = a.p.n_kv * a.ngrp;
    u64 before, u;
    if (a.n_seqs <= 64) {
        const int i = lane < a.n_seqs ? lane : a.n_seqs - 1;
        const Seq q = seq_of(a, a.cu[i], a.cu[i + 1], a.lens[i]);
        const u64 mine = lane < a.n_seqs && q.n ? items_measure(a, q, seq_items(a, q)) : 0, x = wave_scan(mine);
        line = line_of(a, lane_u64(x, 63) * rep);
        u = at(line);
        const u64 past = __ballot(x * rep > u);
        if (!past) return false;
        o.s = __builtin_ctzll(past);
        before = lane_u64(x - mine, o.s);
        o.q.r0 = __builtin_amdgcn_readlane(q.r0, o.s);
        o.q.n = __builtin_amdgcn_readlane(q.n, o.s);
        o.q.hist = __builtin_amdgcn_readlane(q.hist, o.s);
    } else {
        constexpr int NWV = NT / 64;
        const int per = (a.n_seqs + NT - 1) / NT, s0 = tid * per;
        auto measure = [&](int s) {
            const Seq q = seq_of(a, a.cu[s], a.cu[s + 1], a.lens[s]);
            return q.n ? items_measure(a, q, seq_items(a, q)) : (u64)0;
        };
        u64 sum = 0;
        for (int i = 0; i < per; i++)
            if (s0 + i < a.n_seqs) sum += measure(s0 + i);
        const u64 x = wave_scan(sum);
        if (lane == 63) red[wave] = x;
        if (tid == 0) red[NWV] = ~(u64)0;
        lds_sync();
        u64 b = x - sum, all = 0;
#pragma unroll
        for (int w = 0; w < NWV; w++) {
            if (w < wave) b += red[w];
            all += red[w];
        }
        line = line_of(a, all * rep);
        u = at(line);
        if (u >= b * rep && u < (b + sum) * rep) {
            int s = s0;
            for (;; s++) {
                const u64 v = measure(s);
                if (u < (b + v) * rep) break;
                b += v;
            }
            red[NWV] = b;
            red[NWV + 1] = (unsigned)s;
        }
        lds_sync();
        before = red[NWV];
        if (before == ~(u64)0) return false;
        o.s = __builtin_amdgcn_readfirstlane((int)red[NWV + 1]);
        before = lane_u64(before, 0);
        o.q = seq_of(a, a.cu[o.s], a.cu[o.s + 1], a.lens[o.s]);
        lds_sync();
    }
    const int items = seq_items(a, o.q);
    const u64 one = items_measure(a, o.q, items), off = u - before * rep;
    // the quotient, whose double is off by one at most
    int r = (int)((double)off / (double)one);
    if ((u64)r * one > off) r--;
    else if ((u64)(r + 1) * one <= off) r++;
    o.rep = __builtin_amdgcn_readfirstlane(r);
    const u64 y = off - (u64)o.rep * one;
    // the last item that begins at y or before: 64 candidates a step
    int lo = 0, n = items;
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const bool in = (long)lane * step < n && items_measure(a, o.q, lo + lane * step) <= y;
        const int c = __popcll(__ballot(in));
        lo += (c > 0 ? c - 1 : 0) * step;
        n = items - lo < step ? items - lo : step;
    }
    o.item = __builtin_amdgcn_readfirstlane(lo);
    o.x = lane_u64(y - items_measure(a, o.q, o.item), 0);
    o.size = lane_u64(item_measure(a, o.q, o.item), 0);
    return true;
}

// an item's rows, keys and 32-key tiles
struct Item {
    int row0, rows, kfirst, klast, kt0, tiles;
    __device__ __forceinline__ Item(const ChunkArgs& a, const Place& p) {
        row0 = p.item * a.rpi;
        rows = p.q.n - row0 < a.rpi ? p.q.n - row0 : a.rpi;
        kfirst = first_key(a, p.q.hist + row0);
        klast = p.q.hist + row0 + rows - 1;
        kt0 = kfirst >> 5;
        tiles = (klast >> 5) - kt0 + 1;
    }
    // the tile that a share which begins at x of the item begins with
    __device__ __forceinline__ int tile_at(u64 x, u64 size) const {
        if (x >= size) return tiles;
        const int t = (int)((kfirst + (x > kLead ? x - kLead : 0)) >> 5) - kt0;
        return t < tiles ? t : tiles;
    }
};
// What the second launch has to know of a share, at the head of part; the place
// in out is that of the item which the share has from the one before it.
enum : unsigned {
    kGoesIn = 1,      // the share's first item began before it
    kTilesIn = 2,     // and has tiles in it,
    kFromTile0 = 4,   // its first among them;
    kGoesThrough = 8, // and goes on behind it
    kGoesOut = 16,    // an item that begins in the share goes on behind it
    kTilesOut = 32,   // and has tiles in it
    kColsShift = 8,   // columns of the first item, at most 128
};
struct ShareNote {
    int row, nh, head;   // first row of out, heads, first head
};
struct Notes {
    unsigned flags[kShares];
    ShareNote item[kShares];
};
// floats of a partial result: 32 columns at a time in the order of a wave's
// registers, then each column's maximum and weight sum (head_dim 512: for each
// half of the dims, whose V rows have exponents of their own)
__host__ __device__ inline size_t part_floats(int cols, int hd) { return (size_t)cols * (hd + 4); }

// ---- types ----------------------------------------------------------------------
// TQ: rows, TC: cache.  NQ, NK, NP: terms of q, of K (and V), of the weights.
// REG: tiles go through registers, where they are put into other numbers
// (codes into bf16, fp32 into halves); the others go from the pages to LDS.
template <int TQ, int TC>
struct Mode {
    static constexpr int ES = TC == G4_F32 ? 4 : TC == G4_KV_Q8 ? 1 : 2;
    static constexpr bool kHalf = TC == G4_F32 || TC == G4_F16;     // fp16 operands
    static constexpr bool F = TC == G4_F32, Q8 = TC == G4_KV_Q8, REG = F || Q8;
    static constexpr int NQ = TQ != G4_F32 ? 1 : kHalf ? 2 : 3, NK = F ? 2 : 1, NP = NQ;
    // a score is the sum of products as it stands, times log2(e) scale
    static constexpr bool kRaw = !F && !Q8 && NQ < 3;
    // rows of O^T are its dims, in 16 bits pairs of dims 16 apart
    static constexpr bool kPairs = !REG;
    // how far a score may pass the maximum before it moves, and how far above the
    // largest score it is put.  bf16, whose V goes as far as fp32: weights are at
    // most 1; fp16's smallest numbers ask for large weights, and its V cannot overflow
    static constexpr float kSlack = !kHalf ? 0.0f : NQ == 1 ? 8.0f : 4.0f, kRaise = kHalf ? 0.0f : 8.0f;
    // fp16 weights and terms: 2^7 and 2^11 above their fp32 size, with kSlack 2^15 at most.
    // Half of fp16's smallest step is then 2^-32 (2^-36) of the largest weight: a long tail
    // of small ones keeps its share
    static constexpr float kLift = !kHalf ? 0.0f : NQ == 1 ? 7.0f : 11.0f;
};
template <int T>
struct RowElem;
template <>
struct RowElem<G4_F32> { typedef float t; };
template <>
struct RowElem<G4_F16> { typedef _Float16 t; };
template <>
struct RowElem<G4_BF16> { typedef __bf16 t; };
template <bool HALF>
struct OpOf { typedef b8_t t; };
template <>
struct OpOf<true> { typedef h8_t t; };

// A wave's job is 32 columns (row, q head) of an item; a workgroup's jobs share
// its tiles of 32 keys in LDS.  S^T = K Q^T (rows keys, columns q rows): a lane
// holds 16 of a column's 32 scores, which are, as they stand, its operand of
// O^T += V^T P^T.  The cache's blocks have their operands' order, so that 16-bit
// tiles go from the pages to LDS as they are.  The running maximum moves only
// when a score passes it by kSlack.
//   16 bits, head_dim up to 256: eight waves, KSP 2: the two waves of a SIMD have the
// same job and every other tile, waves 4 .. 7 their second product a tile later.
//   16 bits, 512: four waves, q (128) and o (256) in one wave's 512 registers.  (Dims
// halved over two of eight waves, whose partial scores met in LDS: 512 rows over
// 32488 positions 393 us against 366.)
//   q of several terms, and codes: four waves; 512, terms: DS 2, the dims halved over
// two waves, whose partial scores meet in LDS.
// 8 heads on 2 kv heads, the whole call, in a row over the same buffers (behind it with
// others each time): 512 rows over 32488 positions, bf16 of 512, 316 us (335), 870 TFLOP/s
// where an 8192^3 library product reaches 1204; there LDS is read for 45 % of the cycles,
// the matrix cores are busy for 44 %.  fp32 over fp16 of 256 (two products each), 1470
// rows over 4700 positions 142 us (143), 430 of them (865 with the second terms).  fp32 of
// 512, 250 rows over 16001, 328 us (337), 200 (600): a wave's instructions bound it, 1100
// a tile for splitting K and V into halves (640) and for the weights, against 96 products
// of 32 cycles.
template <int TQ, int TC, int HD>
struct Plan {
    typedef Mode<TQ, TC> M;
    static constexpr int DS = HD == 512 && M::NQ > 1 ? 2 : 1;
    static constexpr int NW = M::NQ == 1 && !M::REG && HD < 512 ? 8 : 4;   // waves; 8: two a SIMD
    static constexpr int KSP = NW == 8 && DS == 1 ? 2 : 1;           // tiles at a time
    static constexpr int NJ = NW / DS / KSP, COLS = 32 * NJ;
    // LDS: K and V of a tile are TB bytes each
    static constexpr int TB = 64 * HD * M::NK;
    static constexpr bool ONE = DS == 2 && M::REG;                   // one place each for K and V
    static constexpr int NKP = ONE ? 1 : 2 * KSP, NVP = ONE ? 1 : KSP == 2 ? 5 : 2;
    // staging: a wave has a 16-token block of K or V, KC kilobytes.  BOTH: half of the
    // dims of a block of K and of one of V instead
    static constexpr int KC = HD * M::ES / 64;
    static constexpr bool BOTH = M::REG && NW == 4 && KC > 1;
    static constexpr int PH = BOTH ? KC / 2 : 1;
    static constexpr int MB = BOTH ? 1024 : 512;                     // a tile's factors and marks
    static constexpr int META = (NKP + NVP) * TB, TOPX = META + 2 * KSP * MB, XCH = TOPX + (BOTH ? 256 : 0);
    static constexpr int RB = HD / DS * (TQ == G4_F32 ? 4 : 2);      // bytes of a wave's part of a row
    static constexpr int END = XCH + (DS == 2 ? 16384 : 0);          // DS 2: partial scores
    static constexpr int ROWS = (KSP == 1 ? NW : 0) * 32 * RB;       // the output's rows
    static constexpr int JOIN = KSP == 2 ? NJ * (HD * 128 + 256) : 0;   // sums of waves 4 .. 7
    static constexpr int TOP0 = END > ROWS ? END : ROWS, TOP = TOP0 > JOIN ? TOP0 : JOIN;
    static constexpr int RED = (TOP + 15) / 16 * 16, LDS = RED + 128;
    static_assert(LDS <= 160 * 1024 && NJ * DS * KSP == NW, "LDS");
    static_assert((BOTH || NW == 4 * KSP) && (!BOTH || PH * 2 == KC), "pieces");
    static __device__ __forceinline__ int k_at(int st, int kp) { return ONE ? 0 : ((st & 1) * KSP + kp) * TB; }
    static __device__ __forceinline__ int v_at(int st, int kp) {
        return (NKP + (ONE ? 0 : kp == 0 ? st & 1 : 2 + st % 3)) * TB;
    }
    static __device__ __forceinline__ int meta_at(int st, int kp) { return META + ((st & 1) * KSP + kp) * MB; }
};
// What lies beside a tile: 32 factors of K (fp32: 2^e, codes: scales), 32 of V
// (exponents, scales), fp32: 2^-e; marks of each block's keys that make a score
// NaN.  BOTH: K's, V's and the inverses for each half of the dims, 32 each, marks
// of K and V for each block and half.
constexpr int kMetaV = 128, kMetaMarks = 384;
constexpr int kBothV = 256, kBothInv = 512, kBothMarks = 768;

// SMALL: bf16 rows under a scale below 1.  They go as far as fp32, and their products
// with the keys may pass it where the scale makes ordinary scores of them: the rows take
// the scale's power of two with them (exact but for what becomes subnormal, 2^-134).  8
// heads, this and a.fq alone: 512 rows over 32488 positions, bf16 of 512, 313 us and 300,
// 48 single rows 75 and 71; 23 rows of 256 24.3 and 23.7.  A kernel of its own: as a
// branch of one kernel it cost the other scales up to 4 % (512 rows 317 -> 329).
template <int TQ, int TC, int HD, bool SMALL>
__global__ __launch_bounds__((64 * Plan<TQ, TC, HD>::NW), (Plan<TQ, TC, HD>::NW / 4)) void attn_chunk_kernel(ChunkArgs a) {
    typedef Plan<TQ, TC, HD> P;
    typedef Mode<TQ, TC> M;
    typedef typename RowElem<TQ>::t E;
    typedef typename OpOf<M::kHalf>::t op;
    constexpr int NW = P::NW, DS = P::DS, NJ = P::NJ, KSP = P::KSP, TB = P::TB, KC = P::KC;
    constexpr int NQ = M::NQ, NK = M::NK, NP = M::NP, ES = M::ES;
    constexpr int KS = HD / 16 / DS, NT = HD / 32 / DS;   // a wave's product steps and 32-dim tiles
    extern __shared__ __align__(16) uint8_t lds[];
    u64* red = reinterpret_cast<u64*>(lds + P::RED);
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), part = wave % DS, kp = wave / (NJ * DS), slot = wave / DS % NJ;
    // this wave's share of the staging: tile of a stage, K or V, block of the tile
    const int ut = wave >> 2, uv = wave >> 1 & 1, ub = wave & 1;

    Line line;
    Place at;
    unsigned share = 0;
    Notes* const notes = reinterpret_cast<Notes*>(a.part);
    if (!find_place<64 * NW>(
            a,
            [&](const Line& l) {
                // neighbours on the line, which look at the same keys, to one XCD
                share = l.lg == kLgShares ? (blockIdx.x & 7) * (kShares / 8) + (blockIdx.x >> 3) : blockIdx.x;
                return share >> l.lg ? kNowhere : l.at(share);
            },
            line, at, red)) {
        if (tid == 0) notes->flags[share] = 0;
        return;
    }
    u64 left = line.at(share + 1) - line.at(share);
    unsigned note = at.x > 0 ? kGoesIn : 0;
    ShareNote noted = {};

    while (left > 0) {
        const u64 take = left < at.size - at.x ? left : at.size - at.x;
        const Item it(a, at);
        const int tile0 = it.tile_at(at.x, at.size), tile1 = it.tile_at(at.x + take, at.size);
        const bool goes_on = at.x + take < at.size;
        if (at.x > 0) {
            const int kvh = at.rep / a.ngrp, hg = at.rep - kvh * a.ngrp;
            note |= (tile0 < tile1 ? kTilesIn : 0) | (tile0 == 0 ? kFromTile0 : 0) | (goes_on ? kGoesThrough : 0);
            noted.row = at.q.r0 + it.row0;
            noted.nh = a.group - hg * a.gh < a.gh ? a.group - hg * a.gh : a.gh;
            noted.head = kvh * a.group + hg * a.gh;
            note |= (unsigned)(it.rows * noted.nh) << kColsShift;
        } else if (goes_on) {
            note |= kGoesOut | (tile0 < tile1 ? kTilesOut : 0);
        }
        if (tile0 < tile1) {
            // every part of an item's work has a lane number of its own, so that no
            // address derived from it is kept in a register over the others
            auto own_lane = [&]() {
                int x = tid & 63;
                asm volatile("" : "+v"(x));
                return x;
            };
            const int lane = own_lane(), t16 = lane & 15, g = lane >> 4;
            const int kvh = at.rep / a.ngrp, hg = at.rep - kvh * a.ngrp;
            const int nh = a.group - hg * a.gh < a.gh ? a.group - hg * a.gh : a.gh;    // heads there are
            const int head0 = kvh * a.group + hg * a.gh;
            const int ncols = it.rows * nh;
            const bool mine = slot * 32 < ncols;
            // column j: row j / nh, head j % nh; columns past the last repeat it
            const unsigned inv_nh = (65535u + nh) / (unsigned)nh;   // j < 128: j / nh exactly
            auto col_row = [&](int j, int& hh) {
                j = j < ncols ? j : ncols - 1;
                const int r = (int)((unsigned)j * inv_nh >> 16);
                hh = j - r * nh;
                return it.row0 + r;
            };
            int unused;
            // tiles that every column of the job sees whole: full0 .. full1
            const int jfirst = at.q.hist + col_row(slot * 32, unused), jlast = at.q.hist + col_row(slot * 32 + 31, unused);
            const int full0 = (first_key(a, jlast) + 31) >> 5, full1 = ((jfirst + 1) >> 5) - 1;
            const int ktb = it.kt0 + tile0;                          // the piece's first tile
            const int ntile = tile1 - tile0, stages = (ntile + KSP - 1) / KSP;

            // ---- tiles on their way into LDS: stage st has the tiles ktb + KSP st + (0 .. KSP - 1) ----
            // The page of this wave's block of a stage, -1: not a page, -2: nobody looks
            // at it.  It is asked for a stage ahead: waiting for it would mean waiting
            // for every load before it.
            auto page_in_pool = [&](int asked_page, bool asked) {
                const int p = __builtin_amdgcn_readfirstlane(asked_page);
                return !asked ? -2 : p >= 0 && p < a.p.n_pages ? p : -1;
            };
            int asked_page = 0;
            bool asked = false;
            auto ask_page = [&](int st) {
                const int t = st * KSP + ut, key = (ktb + t) * 32 + ub * 16;
                asked = t < ntile && key + 15 >= it.kfirst && key <= it.klast;
                if (asked) asked_page = a.p.table[(size_t)at.s * a.p.table_stride + (key >> a.p.lgpage)];
            };
            auto block_at = [&](int st, int pg) {
                return a.p.block_of(pg < 0 ? 0 : pg, kvh, (ktb + st * KSP + ut) * 32 + ub * 16);
            };
            auto block_rsrc = [&](size_t block, int pg) {
                return __builtin_amdgcn_make_buffer_rsrc((void*)((uv ? a.p.vp : a.p.kp) + block * (16 * HD * ES)), 0,
                                                         pg < 0 ? 0 : 16 * HD * ES, kBufWord3);
            };
            // tokens of the block from key on that somebody looks at, as bits
            auto tokens_seen = [&](int key) {
                unsigned u = 0xffffu;
                if (it.kfirst > key) u &= it.kfirst - key < 16 ? 0xffffu << (it.kfirst - key) : 0u;
                if (it.klast < key + 15) u &= it.klast >= key ? 0xffffu >> (15 - (it.klast - key)) : 0u;
                return u;
            };
            auto block_use = [&](int st) { return tokens_seen((ktb + st * KSP + ut) * 32 + ub * 16); };
            uint8_t* const mine_meta = lds + kMetaMarks + ub * 4;
            // straight to LDS (K or V, as this wave has it)
            __amdgpu_buffer_rsrc_t copy_rsrc;
            uint8_t* copy_to = lds;
            auto copy_piece = [&](int i) { buf_load_lds16(copy_rsrc, copy_to + i * 1024, (tid & 63) * 16, i * 1024); };
            auto begin_copy = [&](int st) {
                const int pg = page_in_pool(asked_page, asked);
                copy_rsrc = block_rsrc(block_at(st, pg), pg);
                copy_to = lds + (uv ? P::v_at(st, ut) : P::k_at(st, ut)) + ub * KC * 1024;
                if (uv && lane == 0) *reinterpret_cast<unsigned*>(mine_meta + P::meta_at(st, ut)) = pg == -1 ? 0xffffu : 0u;
                ask_page(st + 1);
            };
            auto copy = [&](int st) {
                begin_copy(st);
#pragma unroll
                for (int i = 0; i < KC; i++) copy_piece(i);
            };
            // one wave a SIMD: copies are issued between the products
            constexpr bool kFeed = !M::REG && NW == 4;
            // through registers
            uint4 raw[M::REG ? KC : 1];
            float raw_scale = 0.0f;
            int raw_pg = 0;
            auto fetch = [&](int st) {
                const int pg = page_in_pool(asked_page, asked);
                const size_t block = block_at(st, pg);
                const __amdgpu_buffer_rsrc_t r = block_rsrc(block, pg);
#pragma unroll
                for (int i = 0; i < KC; i++) raw[i] = buf_load16(r, lane * 16, i * 1024);
                if (M::Q8) raw_scale = reinterpret_cast<const float*>((uv ? a.p.vp : a.p.kp) + a.p.scale_off)[block * 16 + t16];
                raw_pg = pg;
                ask_page(st + 1);
            };
            // 16 codes as bf16
            auto codes8 = [&](const uint4& x, unsigned (&y)[8]) {
                const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int c0 = (int8_t)(w[k >> 1] >> (k & 1 ? 16 : 0)), c1 = (int8_t)(w[k >> 1] >> (k & 1 ? 24 : 8));
                    y[k] = hi_halves(__float_as_uint((float)c0), __float_as_uint((float)c1));
                }
            };
            auto put = [&](int st) {
                uint8_t* to = lds + (uv ? P::v_at(st, ut) : P::k_at(st, ut));
                float* meta = reinterpret_cast<float*>(lds + P::meta_at(st, ut));
                const unsigned use = block_use(st);
                unsigned marks = raw_pg == -1 ? 0xffffu : 0u;
                if constexpr (M::Q8) {
                    const bool on = use >> t16 & 1 && raw_pg >= 0;
                    // scales that are not finite: of heads with infinities or NaN
                    const bool bad = on && !(fabsf(raw_scale) < INFINITY);
                    marks |= (unsigned)__ballot(bad && g == 0) & 0xffffu;
                    if (g == 0) meta[(uv ? kMetaV / 4 : 0) + ub * 16 + t16] = on && !bad ? raw_scale : 0.0f;
#pragma unroll
                    for (int i = 0; i < KC; i++) {
                        const int c = i;
                        unsigned y[8];
                        codes8(raw[i], y);
                        if (uv) {
                            // dims 64 c + 16 k + t16 of tokens 4 g .. 4 g + 3
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                *reinterpret_cast<uint2*>(to + ((2 * c + (k >> 1)) * 2 + ub) * 1024 +
                                                          ((g & 1) * 32 + (k & 1) * 16 + t16) * 16 + (g >> 1) * 8) =
                                    make_uint2(y[2 * k], y[2 * k + 1]);
                        } else {
                            // dims 64 c + 16 g .. + 15 of token t16
#pragma unroll
                            for (int k = 0; k < 2; k++)
                                *reinterpret_cast<uint4*>(to + (4 * c + g) * 1024 + (k * 32 + ub * 16 + t16) * 16) =
                                    make_uint4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
                        }
                    }
                }
                // K's and V's marks have a word each: [K or V][block]
                if (lane == 0) reinterpret_cast<unsigned*>(meta)[kMetaMarks / 4 + (uv ? 0 : 4) + ub] = marks;
            };

            // BOTH: half hf of the dims of block bb, K and V.  A piece is put into LDS
            // between the products and its registers take the next tile's at once.
            constexpr int PH = P::PH;
            constexpr bool BOTH = P::BOTH;
            const int bb = wave & 1, hf = wave >> 1;
            uint4 rk[BOTH ? PH : 1], rv[BOTH ? PH : 1];
            float ks16 = 0.0f, vs16 = 0.0f, sfk = 0.0f, sfv[4];
            int askk = 0, askv = 0, pgk = -2, pgv = -2;     // page asked for; page of what the registers hold
            bool onk = false, onv = false;
            __amdgpu_buffer_rsrc_t nk, nv;
            auto ask2 = [&](int st, int& page, bool& on) {
                const int key = (ktb + st) * 32 + bb * 16;
                on = st < ntile && key + 15 >= it.kfirst && key <= it.klast;
                if (on) page = a.p.table[(size_t)at.s * a.p.table_stride + (key >> a.p.lgpage)];
            };
            auto use2 = [&](int st) { return tokens_seen((ktb + st) * 32 + bb * 16); };
            // stage st's page looked up: its loads may follow
            auto open2 = [&](int st, bool v) {
                const int pg = v ? page_in_pool(askv, onv) : page_in_pool(askk, onk);
                const size_t block = a.p.block_of(pg < 0 ? 0 : pg, kvh, (ktb + st) * 32 + bb * 16);
                const uint8_t* pool = v ? a.p.vp : a.p.kp;
                const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(pool + block * (16 * HD * ES)), 0,
                                                                                   pg < 0 ? 0 : 16 * HD * ES, kBufWord3);
                float sc16 = 0.0f;
                if (M::Q8) sc16 = reinterpret_cast<const float*>(pool + a.p.scale_off)[block * 16 + t16];
                if (v) {
                    nv = r;
                    pgv = pg;
                    vs16 = sc16;
                    ask2(st + 1, askv, onv);
                } else {
                    nk = r;
                    pgk = pg;
                    ks16 = sc16;
                    ask2(st + 1, askk, onk);
                }
            };
            auto load2 = [&](bool v, int j) {
                const uint4 x = buf_load16(v ? nv : nk, hf * PH * 1024 + lane * 16, j * 1024);
                if (v) rv[j] = x;
                else rk[j] = x;
            };
            // largest of two numbers and one that is positive or NaN, which it stays
            auto larger = [](uint32_t x, uint32_t y, float top) {
                return __builtin_elementwise_maximum(__builtin_elementwise_maximum(fabsf(__uint_as_float(x)), fabsf(__uint_as_float(y))), top);
            };
            // before the pieces of stage st, which the registers hold: factors, marks, and
            // the next stage's page
            auto begin_k = [&](int st) {
                float* meta = reinterpret_cast<float*>(lds + P::meta_at(st, 0));
                const unsigned use = use2(st);
                unsigned marks = pgk == -1 ? 0xffffu : 0u;
                if constexpr (M::F) {
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < PH; i++) {
                        top = larger(rk[i].x, rk[i].y, top);
                        top = larger(rk[i].z, rk[i].w, top);
                    }
#pragma unroll
                    for (int d = 16; d < 64; d <<= 1) top = __builtin_elementwise_maximum(top, shfl_xor(top, d));
                    const bool bad = !(top < INFINITY);
                    int e = (int)(__float_as_uint(top) >> 23);
                    if (bad || e < kLowK) e = kLowK;
                    marks |= (unsigned)__ballot(bad && g == 0 && (use >> t16 & 1)) & 0xffffu;
                    sfk = row_scale(e);
                    if (g == 0) meta[hf * 32 + bb * 16 + t16] = row_scale_inv(e);
                } else {
                    const bool on = use >> t16 & 1 && pgk >= 0, bad = on && !(fabsf(ks16) < INFINITY);
                    marks |= (unsigned)__ballot(bad && g == 0) & 0xffffu;
                    if (g == 0 && hf == 0) meta[bb * 16 + t16] = on && !bad ? ks16 : 0.0f;
                }
                if (lane == 0) reinterpret_cast<unsigned*>(meta)[kBothMarks / 4 + hf * 2 + bb] = marks;
                open2(st + 1, false);
            };
            // V, fp32: each token's largest, of this half of the dims
            auto tops_v = [&](float (&top)[4]) {
#pragma unroll
                for (int k = 0; k < 4; k++) top[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < PH; i += 2) {
                    top[0] = larger(rv[i].x, rv[i + 1].x, top[0]);
                    top[1] = larger(rv[i].y, rv[i + 1].y, top[1]);
                    top[2] = larger(rv[i].z, rv[i + 1].z, top[2]);
                    top[3] = larger(rv[i].w, rv[i + 1].w, top[3]);
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    top[k] = __builtin_elementwise_maximum(top[k], dpp_f<kDppXor1>(top[k]));
                    top[k] = __builtin_elementwise_maximum(top[k], dpp_f<kDppXor2>(top[k]));
                    top[k] = __builtin_elementwise_maximum(top[k], dpp_f<kDppHalfMirror>(top[k]));
                    top[k] = __builtin_elementwise_maximum(top[k], dpp_f<kDppMirror>(top[k]));
                }
            };
            float* const topx = reinterpret_cast<float*>(lds + P::TOPX);
            auto share_tops = [&]() {
                float top[4];
                tops_v(top);
                if (t16 == 0) *reinterpret_cast<f4_t*>(topx + hf * 32 + bb * 16 + 4 * g) = f4_t{top[0], top[1], top[2], top[3]};
            };
            auto begin_v = [&](int st) {
                float* meta = reinterpret_cast<float*>(lds + P::meta_at(st, 0));
                const unsigned use = use2(st);
                unsigned marks = pgv == -1 ? 0xffffu : 0u;
                if constexpr (M::F) {
                    float top[4];
                    if constexpr (DS == 1) {
                        // a token's weight carries one exponent, whichever the dim
                        const f4_t x = *reinterpret_cast<const f4_t*>(topx + bb * 16 + 4 * g);
                        const f4_t y = *reinterpret_cast<const f4_t*>(topx + 32 + bb * 16 + 4 * g);
#pragma unroll
                        for (int k = 0; k < 4; k++) top[k] = __builtin_elementwise_maximum(x[k], y[k]);
                    } else {
                        tops_v(top);
                    }
                    float ex[4];
                    bool odd = false;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const bool on = use >> (4 * g + k) & 1, bad = !(top[k] < INFINITY);
                        int e = (int)(__float_as_uint(top[k]) >> 23);
                        if (bad || !on || e < kLowV) e = kLowV;
                        odd = odd || bad || !on;
                        sfv[k] = row_scale(e);
                        ex[k] = on ? (float)(e - 141) : 113.0f;     // of no weight: not the smallest
                    }
                    if (__any(odd)) {
                        // rows that are not finite, or that nobody looks at, become zeros
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const bool on = use >> (4 * g + k) & 1, bad = !(top[k] < INFINITY);
                            const u64 b = __ballot(on && bad && t16 == 0);   // lanes 0, 16, 32, 48: tokens k, 4 + k, ..
#pragma unroll
                            for (int j = 0; j < 4; j++) marks |= (unsigned)(b >> (16 * j) & 1) << (4 * j + k);
                            if (bad || !on) {
#pragma unroll
                                for (int i = 0; i < PH; i++) {
                                    if (k == 0) rv[i].x = 0;
                                    else if (k == 1) rv[i].y = 0;
                                    else if (k == 2) rv[i].z = 0;
                                    else rv[i].w = 0;
                                }
                            }
                        }
                    }
                    if (t16 == 0) {
                        const int to = hf * 32 + bb * 16 + 4 * g;
                        *reinterpret_cast<f4_t*>(meta + kBothV / 4 + to) = f4_t{ex[0], ex[1], ex[2], ex[3]};
                        *reinterpret_cast<f4_t*>(meta + kBothInv / 4 + to) = f4_t{sfv[0], sfv[1], sfv[2], sfv[3]};
                    }
                } else {
                    const bool on = use >> t16 & 1 && pgv >= 0, bad = on && !(fabsf(vs16) < INFINITY);
                    marks |= (unsigned)__ballot(bad && g == 0) & 0xffffu;
                    if (g == 0 && hf == 0) meta[kBothV / 4 + bb * 16 + t16] = on && !bad ? vs16 : 0.0f;
                }
                if (lane == 0) reinterpret_cast<unsigned*>(meta)[kBothMarks / 4 + 4 + hf * 2 + bb] = marks;
                open2(st + 1, true);
            };
            // piece j of stage st to LDS, and the next stage's on its way
            auto piece_k = [&](int st, int j) {
                const int c = hf * PH + j;
                uint8_t* to = lds + P::k_at(st, 0);
                if constexpr (M::F) {
                    h2v_t hi[2], lo[2];
                    split2(__uint_as_float(rk[j].x), __uint_as_float(rk[j].y), sfk, hi[0], lo[0]);
                    split2(__uint_as_float(rk[j].z), __uint_as_float(rk[j].w), sfk, hi[1], lo[1]);
                    to += c * 1024 + ((g >> 1) * 32 + bb * 16 + t16) * 16 + (g & 1) * 8;
                    *reinterpret_cast<uint2*>(to) = make_uint2(h2_bits(hi[0]), h2_bits(hi[1]));
                    *reinterpret_cast<uint2*>(to + 64 * HD) = make_uint2(h2_bits(lo[0]), h2_bits(lo[1]));
                } else {
                    unsigned y[8];
                    codes8(rk[j], y);
#pragma unroll
                    for (int k = 0; k < 2; k++)
                        *reinterpret_cast<uint4*>(to + (4 * c + g) * 1024 + (k * 32 + bb * 16 + t16) * 16) =
                            make_uint4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
                }
                load2(false, j);
            };
            auto piece_v = [&](int st, int j) {
                const int c = hf * PH + j;
                uint8_t* to = lds + P::v_at(st, 0);
                if constexpr (M::F) {
                    h2v_t hi[2], lo[2];
                    split2(__uint_as_float(rv[j].x), __uint_as_float(rv[j].y), sfv[0], sfv[1], hi[0], lo[0]);
                    split2(__uint_as_float(rv[j].z), __uint_as_float(rv[j].w), sfv[2], sfv[3], hi[1], lo[1]);
                    to += ((c >> 1) * 2 + bb) * 1024 + ((g & 1) * 32 + (c & 1) * 16 + t16) * 16 + (g >> 1) * 8;
                    *reinterpret_cast<uint2*>(to) = make_uint2(h2_bits(hi[0]), h2_bits(hi[1]));
                    *reinterpret_cast<uint2*>(to + 64 * HD) = make_uint2(h2_bits(lo[0]), h2_bits(lo[1]));
                } else {
                    unsigned y[8];
                    codes8(rv[j], y);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        *reinterpret_cast<uint2*>(to + ((2 * c + (k >> 1)) * 2 + bb) * 1024 +
                                                  ((g & 1) * 32 + (k & 1) * 16 + t16) * 16 + (g >> 1) * 8) =
                            make_uint2(y[2 * k], y[2 * k + 1]);
                }
                load2(true, j);
            };
            // pieces that belong to step i of n
            auto pieces = [&](int i, int n, auto&& piece) {
#pragma unroll
                for (int j = 0; j < PH; j++)
                    if (j * n / PH == i) piece(j);
            };

            // ---- q: 32 columns' rows through places in LDS that the first stage leaves free ----
            op q[NQ][KS];
            float fq = NQ == 1 ? a.fq : fabsf(a.scale) * kLog2e;
            constexpr int kBox = KSP == 2 ? TB : DS == 1 ? TB / 2 : TB / 4, kPasses = 32 * P::RB / kBox;
            constexpr int kChunks = P::RB / 16 / kPasses, kSteps = KS / kPasses;
            static_assert(kBox == 32 * kChunks * 16 && kSteps * kPasses == KS, "q");
            uint8_t* box = lds + (KSP == 2 ? (slot < 2 ? 2 + slot : slot == 2 ? 5 : 7) * TB
                                  : DS == 1 ? (wave < 2 ? TB : 2 * TB) + wave * (TB / 2)
                                  : TB + wave * (TB / 4));
            auto q_row = [&](int pass) {
                return [=](int r) {
                    int hh;
                    const int row = col_row(slot * 32 + r, hh);
                    return (const uint8_t*)((const E*)a.q + (size_t)(at.q.r0 + row) * a.q_stride + (size_t)(head0 + hh) * HD +
                                            part * (HD / DS)) + pass * kChunks * 16;
                };
            };
            auto load_q = [&]() {
                const int lane = own_lane(), col = lane & 31, h = lane >> 5;
                auto chunk = [&](int c) { return box + row_slot<kChunks>(col, c); };
                if constexpr (TQ != G4_F32) {
                    const unsigned flip = a.scale < 0.0f ? 0x80008000u : 0u;
                    auto shrink = [&](const f4_t& x) {
                        E e[8];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const unsigned w = __float_as_uint(x[k]);
                            e[2 * k] = (E)(__uint_as_float(w << 16) * a.by);
                            e[2 * k + 1] = (E)(__uint_as_float(w & 0xffff0000u) * a.by);
                        }
                        f4_t y;
                        __builtin_memcpy(&y, e, 16);
                        return y;
                    };
#pragma unroll
                    for (int pass = 0; pass < kPasses; pass++) {
                        if constexpr (SMALL) rows_to_lds<kChunks, 32 / KSP>(box, kp * 16, q_row(pass), lane, shrink);
                        else rows_to_lds<kChunks, 32 / KSP>(box, kp * 16, q_row(pass), lane);
                        if constexpr (KSP == 2) lds_barrier();
#pragma unroll
                        for (int i = 0; i < kSteps; i++) {
                            uint4 x = *reinterpret_cast<const uint4*>(chunk(i * 2 + h));
                            if (a.scale == 0.0f) x = make_uint4(0, 0, 0, 0);
                            x.x ^= flip; x.y ^= flip; x.z ^= flip; x.w ^= flip;
                            q[0][pass * kSteps + i] = __builtin_bit_cast(op, x);
                        }
                    }
                } else if constexpr (NQ == 3) {
                    // times scale log2(e), as three terms: the float itself
                    const float qs = a.scale * kLog2e;
#pragma unroll
                    for (int pass = 0; pass < kPasses; pass++) {
                        rows_to_lds<kChunks, 32>(box, 0, q_row(pass), lane);
#pragma unroll
                        for (int i = 0; i < kSteps; i++) {
                            const float4 x = *reinterpret_cast<const float4*>(chunk(i * 4 + h * 2));
                            const float4 y = *reinterpret_cast<const float4*>(chunk(i * 4 + h * 2 + 1));
                            uint32_t t[4][3];
                            split_pair<3>(x.x * qs, x.y * qs, t[0]);
                            split_pair<3>(x.z * qs, x.w * qs, t[1]);
                            split_pair<3>(y.x * qs, y.y * qs, t[2]);
                            split_pair<3>(y.z * qs, y.w * qs, t[3]);
#pragma unroll
                            for (int k = 0; k < NQ; k++) {
                                const uint4 z = make_uint4(t[0][k], t[1][k], t[2][k], t[3][k]);
                                q[k][pass * kSteps + i] = __builtin_bit_cast(op, z);
                            }
                        }
                    }
                    fq = 1.0f;
                } else {
                    float4 x[KS][2];
                    unsigned top = 0;
#pragma unroll
                    for (int pass = 0; pass < kPasses; pass++) {
                        rows_to_lds<kChunks, 32>(box, 0, q_row(pass), lane);
#pragma unroll
                        for (int i = 0; i < kSteps; i++)
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                const float4 y = *reinterpret_cast<const float4*>(chunk(i * 4 + h * 2 + j));
                                x[pass * kSteps + i][j] = y;
                                const float e[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                                for (int k = 0; k < 4; k++) {
                                    const unsigned b = __float_as_uint(e[k]) & 0x7fffffffu;
                                    top = b > top ? b : top;
                                }
                            }
                    }
                    unsigned o = __shfl_xor(top, 32, 64);
                    top = o > top ? o : top;
                    if constexpr (DS == 2) {
                        // of both halves: the partial scores have to be of one scale
                        unsigned* xch = reinterpret_cast<unsigned*>(lds + P::XCH);
                        xch[wave * 64 + lane] = top;
                        lds_barrier();
                        o = xch[(wave ^ 1) * 64 + lane];
                        top = o > top ? o : top;
                    }
                    const int e = (int)(top >> 23) > kLowK ? (int)(top >> 23) : kLowK;
                    float sf = row_scale(e < 255 ? e : 254);
                    fq *= e < 255 ? row_scale_inv(e) : __uint_as_float(0x7fc00000u);
                    if (a.scale < 0.0f) sf = -sf;
                    if (a.scale == 0.0f) {   // a score of -infinity times fq has to stay one
                        sf = 0.0f;
                        fq = e < 255 ? 1.0f : fq;
                    }
                    // nor may it be 0 by underflow: scores are below 2^40 fq
                    if (M::kRaw && fq < FLT_MIN) fq = FLT_MIN;
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
                }
            };

            // ---- first stage, q ----
            if constexpr (BOTH) {
                ask2(0, askk, onk);
                ask2(0, askv, onv);
                open2(0, false);
                open2(0, true);
#pragma unroll
                for (int j = 0; j < PH; j++) {
                    load2(false, j);
                    load2(true, j);
                }
                load_q();
                if constexpr (DS == 2) lds_barrier();   // the boxes have been read
                if constexpr (DS == 1 && M::F) {
                    share_tops();
                    lds_barrier();
                }
                begin_k(0);
#pragma unroll
                for (int j = 0; j < PH; j++) piece_k(0, j);
                if constexpr (DS == 1) {
                    begin_v(0);
#pragma unroll
                    for (int j = 0; j < PH; j++) piece_v(0, j);
                }
            } else if constexpr (M::REG) {
                ask_page(0);
                fetch(0);
                load_q();
                put(0);
                fetch(1);
            } else {
                ask_page(0);
                copy(0);
                load_q();
            }
            // one wave a SIMD: two terms of q stay in the accumulation registers, from which
            // products take them as well (left to itself the compiler moves them there and
            // back for every tile)
            if constexpr (NW == 4 && NQ > 1 && HD >= 256) {
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int i = 0; i < KS; i++) {
                        asm("" : "+a"(q[k][i]));
                    }
            }
            f16_t o[NT] = {};
            float m = -FLT_MAX, l = 0.0f;
            bool fresh = true;   // no tile has been weighted: o is 0
            f16_t sc;
            op p[NP][2];
            struct Ops {
                op x[NK];
            };
            // a lane's place in a tile
            auto k_place = [&]() {
                const int lane = own_lane(), c = lane & 31;
                return M::REG ? lane * 16 : (c >> 4) * KC * 1024 + (lane >> 5) * 256 + (c & 15) * 16;
            };
            auto v_place = [&]() {
                const int lane = own_lane(), c = lane & 31;
                // row r of a product is dim 16 (r & 1) + r / 2 of its 32: neighbours read
                // neighbours (in the order of the dims, 16 bytes apart, twice the cycles)
                return M::REG ? lane * 16 : (lane >> 5) * 256 + c * 8;
            };
            auto read_k = [&](const uint8_t* from, int i, Ops& k) {
                const int s = part * KS + i;
#pragma unroll
                for (int j = 0; j < NK; j++)
                    k.x[j] = *reinterpret_cast<const op*>(from + (M::REG ? j * 64 * HD + s * 1024 : (s >> 1) * 1024 + (s & 1) * 512));
            };
            auto read_v = [&](const uint8_t* from, int i, Ops& v) {
                const int s = part * NT * 2 + i;
                if constexpr (M::REG) {
#pragma unroll
                    for (int j = 0; j < NK; j++) v.x[j] = *reinterpret_cast<const op*>(from + j * 64 * HD + s * 1024);
                } else {
                    const uint8_t* x = from + (s & 1) * KC * 1024 + (s >> 1) * 1024;
                    const uint2 y = *reinterpret_cast<const uint2*>(x), z = *reinterpret_cast<const uint2*>(x + 512);
                    v.x[0] = __builtin_bit_cast(op, make_uint4(y.x, y.y, z.x, z.y));
                }
            };
            // feed(i): what is done beside step i's products
            auto scores = [&](int st, auto&& feed) {
                const uint8_t* from = lds + P::k_at(st, kp) + k_place();
                sc = f16_t{};
                if constexpr (NW == 8) {
#pragma unroll
                    for (int i = 0; i < KS; i++) {
                        Ops k;
                        read_k(from, i, k);
                        sc = mfma32(k.x[0], q[0][i], sc);
                    }
                    order_products<KS, 3, 1, 1>();
                } else {
                    f16_t sx = {}, low;
                    run_products<Ops, KS, (NQ == 1 ? 6 : NK == 2 ? 2 : 3)>([&](int i, Ops& k) { read_k(from, i, k); },
                                             [&](int i, const Ops& k) {
                                                 sc = mfma32(k.x[0], q[0][i], sc);
                                                 feed(i);
#pragma unroll
                                                 for (int j = 1; j < NQ; j++) sx = mfma32(k.x[0], q[j][i], sx);
                                                 if constexpr (NK == 2) sx = mfma32(k.x[1], q[0][i], sx);
                                                 // fp32: K's scales are those of half of the dims
                                                 if (M::F && DS == 1 && i == KS / 2 - 1) {
                                                     low = sc + sx;
                                                     sc = f16_t{};
                                                     sx = f16_t{};
                                                 }
                                             });
                    if (NQ > 1) sc += sx;
                    if constexpr (M::F) {
                        const float* meta = reinterpret_cast<const float*>(lds + P::meta_at(st, 0));
                        const int h = own_lane() >> 5;
                        // The key's 2^e and the row's fq may be far above 1, one of them where scores
                        // are ordinary: fq comes first if it is below 1, and last (weights) if not,
                        // so that nothing on the way is above both the sum and the score.
                        const float fa = fminf(fq, 1.0f);
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            const f4_t x = *reinterpret_cast<const f4_t*>(meta + (DS == 1 ? 32 : part * 32) + 8 * b + 4 * h);
                            const f4_t y = *reinterpret_cast<const f4_t*>(meta + 8 * b + 4 * h);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                sc[4 * b + i] = sc[4 * b + i] * fa * x[i];
                                if constexpr (DS == 1) sc[4 * b + i] = __builtin_fmaf(low[4 * b + i] * fa, y[i], sc[4 * b + i]);
                            }
                        }
                    }
                }
            };
            auto weights = [&](int st) {
                const int lane = own_lane(), h = lane >> 5;
                const int kt = ktb + st * KSP + kp;
                const float* meta = reinterpret_cast<const float*>(lds + P::meta_at(st, kp));
                const unsigned* mk = reinterpret_cast<const unsigned*>(meta) + kMetaMarks / 4;
                unsigned marks;
                if constexpr (BOTH) {
                    const unsigned* m2 = reinterpret_cast<const unsigned*>(meta) + kBothMarks / 4;
                    // [K, V][half][block]
                    marks = m2[0] | m2[2] | m2[4] | m2[6] | (m2[1] | m2[3] | m2[5] | m2[7]) << 16;
                } else {
                    marks = mk[0] | mk[1] << 16;
                    if (M::REG) marks |= mk[4] | mk[5] << 16;
                }
                marks = __builtin_amdgcn_readfirstlane(marks);
                float fv[16];       // codes: V's scales, fp32: 2^-e
                float low = 113.0f;
                const int vhalf = M::F && DS == 2 ? part * 32 : 0;
                if constexpr (M::REG) {
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const f4_t v = *reinterpret_cast<const f4_t*>(meta + (BOTH ? kBothV / 4 : kMetaV / 4) + vhalf + 8 * b + 4 * h);
                        if constexpr (M::F) {
                            const f4_t vi = *reinterpret_cast<const f4_t*>(meta + kBothInv / 4 + vhalf + 8 * b + 4 * h);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                sc[4 * b + i] = __builtin_fmaf(sc[4 * b + i], fq < 1.0f ? 1.0f : fq, v[i]);
                                fv[4 * b + i] = vi[i];
                                low = fminf(low, v[i]);
                            }
                        } else {
                            const f4_t k = *reinterpret_cast<const f4_t*>(meta + 8 * b + 4 * h);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                sc[4 * b + i] *= NQ == 3 ? k[i] : fq * k[i];
                                fv[4 * b + i] = v[i];
                            }
                        }
                    }
                }
                if (marks) {
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (marks >> (8 * (r >> 2) + 4 * h + (r & 3)) & 1) sc[r] = __uint_as_float(0x7fc00000u);
                }
                if (kt < full0 || kt > full1) {
                    const int pos = at.q.hist + col_row(slot * 32 + (lane & 31), unused);
                    const int hi = pos - kt * 32 - 4 * h, lo = first_key(a, pos) - kt * 32 - 4 * h;
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int key = 8 * (r >> 2) + (r & 3);
                        if (key > hi || key < lo) sc[r] = -INFINITY;
                    }
                }
                float top = sc[0];
#pragma unroll
                for (int r = 1; r < 16; r++) top = fmaxf(top, sc[r]);
                if constexpr (M::kRaw) top *= fq;
                // The maximum moves for all of a wave's columns at once, so that what one of
                // them sees decides how the others' weights are rounded.  (Each by itself,
                // with the same bits whatever the others see, moves more often: 512 rows
                // over 32488 positions, bf16 of 512, 316 -> 333 us, over 16000 of codes 222
                // -> 244, 1470 rows over fp32, fp16 and bf16 of 256 1 to 3 %.)
                if (__any(top > m + M::kSlack)) {
                    top = fmaxf(top, shfl_xor(top, 32));
                    top = fmaxf(top + M::kRaise, m);
                    const float f = exp2f(m - top);
                    if constexpr (M::F) l = move_sum(l, m - top);
                    else l *= f;
                    m = top;
                    // (also where l is 0 by now: the factor may have taken all of it)
                    if (!fresh) {
#pragma unroll
                        for (int i = 0; i < NT; i++) o[i] *= f;
                    }
                }
                fresh = false;
                const float base = m - M::kLift;
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    float w[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float x = sc[8 * t + j];
                        w[j] = __builtin_amdgcn_exp2f(M::kRaw ? __builtin_fmaf(x, fq, -base) : x - base);
                        if constexpr (M::F) l = __builtin_fmaf(w[j], fv[8 * t + j], l);
                        else l += w[j];
                        if constexpr (M::Q8) w[j] *= fv[8 * t + j];
                    }
                    if constexpr (NP == 1) {
                        // Rounded to the type, the operand's, while l keeps fp32: 512 rows over
                        // 32488 positions, bf16 of 512, 313 us with an error of 0.00191 of the
                        // norm, where the output's own rounding alone makes 0.00166; two terms
                        // reach that in 404.  A chunk of 471 rows beside 40 single ones 82 us
                        // (0.00204) and 90, over codes, whose scale is rounded with the weight, 512
                        // rows of 512 over 16000 224 (0.00236) and 253, 1470 of 256 137 (0.00231)
                        // and 153.  fp16 of 512 and of 256: 0.000242 and 0.000247 where its own
                        // rounding makes 0.000208.
#pragma unroll
                        for (int j = 0; j < 8; j++) p[0][t][j] = (E)w[j];
                    } else if constexpr (M::kHalf) {
                        h2v_t hi[4], lo[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) split2(w[2 * j], w[2 * j + 1], 1.0f, hi[j], lo[j]);
                        __builtin_memcpy(&p[0][t], hi, 16);
                        __builtin_memcpy(&p[1][t], lo, 16);
                    } else {
                        // three terms: the weight itself (two, each rounded to nearest, are off
                        // by 2^-18 of it: of 169 rows over 39876 positions of codes 2.6e-6 of
                        // the result's norm, 58.8 us against 61.5)
                        uint32_t t3[4][3];
#pragma unroll
                        for (int j = 0; j < 4; j++) split_pair<3>(w[2 * j], w[2 * j + 1], t3[j]);
#pragma unroll
                        for (int k = 0; k < NP; k++) p[k][t] = as_b8(t3[0][k], t3[1][k], t3[2][k], t3[3][k]);
                    }
                }
                if constexpr (M::F) {
                    const float lost = __builtin_ldexpf(1.0f, 48 - 126 - (int)low);   // of this lane's keys
                    if (__any(l < lost)) {
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const int key = 8 * (r >> 2) + 4 * h + (r & 3);
                            l += lost_weight(sc[r] - base, meta[kBothV / 4 + vhalf + key], fv[r]);
                        }
                    }
                }
            };
            auto values = [&](int st, auto&& feed) {
                const uint8_t* from = lds + P::v_at(st, kp) + v_place();
                if constexpr (NW == 8) {
#pragma unroll
                    for (int i = 0; i < 2 * NT; i++) {
                        Ops v;
                        read_v(from, i, v);
                        o[i >> 1] = mfma32(v.x[0], p[0][i & 1], o[i >> 1]);
                    }
                    order_products<2 * NT, 3, 1, 1>();
                } else {
                    run_products<Ops, 2 * NT, (NP == 1 ? 6 : NK == 2 ? 2 : 3)>([&](int i, Ops& v) { read_v(from, i, v); },
                                                 [&](int i, const Ops& v) {
                                                     f16_t& s = o[i >> 1];
                                                     s = mfma32(v.x[0], p[0][i & 1], s);
                                                     feed(i);
#pragma unroll
                                                     for (int k = 1; k < NP; k++) s = mfma32(v.x[0], p[k][i & 1], s);
                                                     if constexpr (NK == 2) s = mfma32(v.x[1], p[0][i & 1], s);
                                                 });
                }
            };
            // Tiles that came straight from the pages: V of tokens that nobody looks at
            // becomes zeros (whatever is there: a weight of 0 times it has to be 0), and
            // where a result was not finite (careful) so do infinities and NaN, whose keys
            // are marked: a column that sees one gets the score NaN, the others what they
            // would have without it, but for rounding (weights).
            auto clean = [&](int st, bool careful) {
                if (M::REG || !uv) return;
                const unsigned use = block_use(st);
                const int lane = own_lane(), g = lane >> 4;
                uint8_t* v = lds + P::v_at(st, ut) + ub * KC * 1024 + lane * 16;
                // this lane's 16 bytes of every piece are two dims of tokens 4 g .. 4 g + 3
                unsigned keep[2], seen = 0;
#pragma unroll
                for (int k = 0; k < 2; k++)
                    keep[k] = (use >> (4 * g + 2 * k) & 1 ? 0xffffu : 0u) | (use >> (4 * g + 2 * k + 1) & 1 ? 0xffff0000u : 0u);
                if (careful) {
#pragma nounroll
                    for (int i = 0; i < KC; i++) {
                        const uint4 x = *reinterpret_cast<const uint4*>(v + i * 1024);
                        unsigned w[4] = {x.x, x.y, x.z, x.w};
                        constexpr unsigned kInf = TC == G4_F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const unsigned sh = 16 * (k & 1);
                            if ((w[k >> 1] >> sh & kInf) == kInf) {
                                w[k >> 1] &= ~(0xffffu << sh);
                                seen |= 1u << (4 * g + (k & 3));
                            }
                        }
                        *reinterpret_cast<uint4*>(v + i * 1024) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    seen &= use;
                    if (seen) atomicOr(reinterpret_cast<unsigned*>(mine_meta + P::meta_at(st, ut)), seen);
                }
#pragma nounroll
                for (int i = 0; i < KC; i++) {
                    uint4 x = *reinterpret_cast<const uint4*>(v + i * 1024);
                    x.x &= keep[0]; x.y &= keep[1]; x.z &= keep[0]; x.w &= keep[1];
                    *reinterpret_cast<uint4*>(v + i * 1024) = x;
                }
            };
            // whether a stage has tokens that nobody looks at
            auto ragged = [&](int st) {
                const int k0 = (ktb + st * KSP) * 32, k1 = (st + 1) * KSP < ntile ? k0 + 32 * KSP - 1 : (ktb + ntile) * 32 - 1;
                return k0 < it.kfirst || k1 > it.klast;
            };

            const auto nothing = [](int) {};
            bool met = false;   // whether all waves have met since their last tile
            for (bool careful = false;; careful = true) {
                if constexpr (BOTH && DS == 1) {
                    for (int st = 0; st < stages; st++) {
                        lds_barrier();   // the stage is there, everyone done with the one before
                        begin_k(st + 1);
                        if (M::F) share_tops();
                        scores(st, [&](int i) { pieces(i, KS, [&](int j) { piece_k(st + 1, j); }); });
                        if (M::F) lds_barrier();   // the largest of V's rows are there
                        begin_v(st + 1);
                        weights(st);
                        values(st, [&](int i) { pieces(i, 2 * NT, [&](int j) { piece_v(st + 1, j); }); });
                    }
                } else if constexpr (BOTH) {
                    f4_t* xch = reinterpret_cast<f4_t*>(lds + P::XCH);
                    for (int st = 0; st < stages; st++) {
                        lds_barrier();   // K is there, V of the tile before done with
                        begin_v(st);
                        scores(st, [&](int i) { pieces(i, KS, [&](int j) { piece_v(st, j); }); });
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            xch[(wave * 4 + i) * 64 + lane] = f4_t{sc[4 * i], sc[4 * i + 1], sc[4 * i + 2], sc[4 * i + 3]};
                        lds_barrier();   // K is done with, the partial scores and V there
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const f4_t y = xch[((wave ^ 1) * 4 + i) * 64 + lane];
#pragma unroll
                            for (int j = 0; j < 4; j++) sc[4 * i + j] += y[j];
                        }
                        begin_k(st + 1);
                        weights(st);
                        values(st, [&](int i) { pieces(i, 2 * NT, [&](int j) { piece_k(st + 1, j); }); });
                    }
                } else {
                    // this wave's copies have landed, then everyone's; and all are done
                    // with the stage before (waves 4 .. 7 but for its V, which has three
                    // places)
                    auto turn = [&](int st) {
                        if constexpr (M::REG) {
                            lds_barrier();
                            if (st + 1 < stages) {
                                put(st + 1);
                                fetch(st + 2);
                            }
                        } else {
                            wait_vm<0>();
                            lds_barrier();
                            if (careful || ragged(st)) {
                                clean(st, careful);
                                lds_barrier();
                            }
                            if (kFeed) begin_copy(st + 1);      // past the last tile: no bytes
                            else if (st + 1 < stages) copy(st + 1);
                        }
                    };
                    auto feed = [&](int i) {
                        if constexpr (kFeed) {
#pragma unroll
                            for (int j = 0; j < KC; j++)
                                if (j * KS / KC == i) copy_piece(j);
                        }
                    };
                    int st = 0;
                    if constexpr (DS == 2) {
                        for (; st < stages; st++) {
                            turn(st);
                            scores(st, feed);
                            // a job's two waves give each other their partial scores
                            const int lane = own_lane();
                            f4_t* xch = reinterpret_cast<f4_t*>(lds + P::XCH) + lane;
                            auto give = [&](int box) {
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    xch[(box * 4 + i) * 64] = f4_t{sc[4 * i], sc[4 * i + 1], sc[4 * i + 2], sc[4 * i + 3]};
                            };
                            f4_t y[4];
                            auto take = [&](int box) {
#pragma unroll
                                for (int i = 0; i < 4; i++) y[i] = xch[(box * 4 + i) * 64];
                            };
                            auto add = [&]() {
#pragma unroll
                                for (int i = 0; i < 4; i++)
#pragma unroll
                                    for (int j = 0; j < 4; j++) sc[4 * i + j] += y[i][j];
                            };
                            give(wave);
                            lds_barrier();
                            take(wave ^ 1);
                            add();
                            weights(st);
                            values(st, nothing);
                        }
                    } else if (KSP == 1 || kp == 0) {
                        for (; st < stages; st++) {
                            turn(st);
                            scores(st, feed);
                            weights(st);
                            values(st, nothing);
                        }
                    } else {
                        turn(st);
                        if (kp < ntile) {
                            scores(st, feed);
                            weights(st);
                        }
                        for (st++; st < stages; st++) {
                            turn(st);
                            values(st - 1, nothing);
                            if (st * KSP + kp < ntile) {
                                scores(st, feed);
                                weights(st);
                            }
                        }
                        if ((stages - 1) * KSP + kp < ntile) values(stages - 1, nothing);
                    }
                }
                // ---- a result that is not finite: once more, carefully ----
                if (M::REG || careful) break;
                float z = 0.0f * l;
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int r = 0; r < 16; r++) z = __builtin_fmaf(0.0f, o[i][r], z);
                unsigned* votes = reinterpret_cast<unsigned*>(red);
                const bool odd = __any(!(z == 0.0f));
                if (lane == 0) votes[wave] = odd;
                wait_vm<0>();
                lds_barrier();
                unsigned any = 0;
#pragma unroll
                for (int w = 0; w < NW; w++) any |= votes[w];
                met = !__builtin_amdgcn_readfirstlane(any);
                if (met) break;
#pragma unroll
                for (int i = 0; i < NT; i++) o[i] = f16_t{};
                m = -FLT_MAX;
                l = 0.0f;
                fresh = true;
                ask_page(0);
                copy(0);
            }

            {
            const int lane = own_lane(), col = lane & 31, h = lane >> 5;
            const bool whole = tile0 == 0 && tile1 == it.tiles;
            l += shfl_xor(l, 32);
            if (!met) {
                wait_vm<0>();
                lds_barrier();
            }
            if constexpr (KSP == 2) {
                // waves 4 .. 7 hand their sums to waves 0 .. 3
                float* ml = reinterpret_cast<float*>(lds + NJ * HD * 128) + slot * 64 + col * 2;
                f4_t* sums = reinterpret_cast<f4_t*>(lds) + slot * HD * 8 + lane;
                if (kp == 1) {
                    if (h == 0) {
                        ml[0] = m;
                        ml[1] = l;
                    }
#pragma unroll
                    for (int i = 0; i < NT; i++)
#pragma unroll
                        for (int b = 0; b < 4; b++)
                            sums[(i * 4 + b) * 64] = f4_t{o[i][4 * b], o[i][4 * b + 1], o[i][4 * b + 2], o[i][4 * b + 3]};
                }
                lds_barrier();
                if (kp == 0) {
                    const float m1 = ml[0], l1 = ml[1], top = fmaxf(m, m1);
                    const float f0 = exp2f(m - top), f1 = exp2f(m1 - top);
                    l = l * f0 + l1 * f1;
                    m = top;
#pragma unroll
                    for (int i = 0; i < NT; i++)
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            const f4_t y = sums[(i * 4 + b) * 64];
#pragma unroll
                            for (int j = 0; j < 4; j++) o[i][4 * b + j] = o[i][4 * b + j] * f0 + y[j] * f1;
                        }
                }
            }
            if (mine && kp == 0) {
                if (whole) {
                    // ---- the output's rows, where K and V (KSP 2: this wave's other sums) were ----
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
                            for (int j = 0; j < 4; j++) y[j] = (E)(o[i][4 * b + (M::kPairs ? (j & 1) * 2 + (j >> 1) : j)] * f);
                            // dims d .. d + 3, or d, d + 1 and 16 more of them
                            constexpr int kTwo = M::kPairs ? 2 : 1;
#pragma unroll
                            for (int k = 0; k < kTwo; k++) {
                                const int d = 32 * i + (M::kPairs ? 16 * k + 4 * b + 2 * h : 8 * b + 4 * h);
                                constexpr int kPer = 16 / sizeof(E), kN = 4 / kTwo * sizeof(E);
                                uint8_t* to = rows + row_slot<kRow>(col, d / kPer) + d % kPer * sizeof(E);
                                __builtin_memcpy(__builtin_assume_aligned(to, kN), y + 4 / kTwo * k, kN);
                            }
                        }
                    rows_from_lds<kRow>(rows, ncols - slot * 32, [&](int r) {
                        int hh;
                        const int row = col_row(slot * 32 + r, hh);
                        return (uint8_t*)((E*)a.out + (size_t)(at.q.r0 + row) * a.out_stride + (size_t)(head0 + hh) * HD +
                                          part * (HD / DS));
                    });
                } else {
                    float* to = a.part + sizeof(Notes) / 4 + (size_t)(share * 2 + (tile0 == 0)) * part_floats(a.cols, HD);
                    f4_t* sums = reinterpret_cast<f4_t*>(to) + (size_t)(slot * DS + part) * NT * 256 + lane;
                    if (slot * 32 + col < ncols) {
#pragma unroll
                        for (int i = 0; i < NT; i++)
#pragma unroll
                            for (int b = 0; b < 4; b++)
                                sums[(i * 4 + b) * 64] = f4_t{o[i][4 * b], o[i][4 * b + 1], o[i][4 * b + 2], o[i][4 * b + 3]};
                        if (h == 0) {
                            float2* ml = reinterpret_cast<float2*>(to + (size_t)a.cols * HD) + slot * 32 + col;
                            ml[part * a.cols] = make_float2(m, l);
                            if (HD == 512 && DS == 1) ml[a.cols] = make_float2(m, l);
                        }
                    }
                }
            }
            }
            lds_barrier();   // LDS is the next item's
        }
        left -= take;
        if (!left) {
            if (tid == 0) {
                notes->flags[share] = note;
                notes->item[share] = noted;
            }
            break;
        }
        // ---- the next item ----
        at.x = 0;
        if (++at.item >= seq_items(a, at.q)) {
            at.item = 0;
            if (++at.rep == a.p.n_kv * a.ngrp) {
                at.rep = 0;
                do {
                    if (++at.s >= a.n_seqs) {   // lengths that changed meanwhile
                        if (tid == 0) notes->flags[share] = 0;
                        return;
                    }
                    at.q = seq_of(a, a.cu[at.s], a.cu[at.s + 1], a.lens[at.s]);
                } while (at.q.n == 0);
            }
        }
        at.size = item_measure(a, at.q, at.item);
    }
}

template <int T>
struct Cached { static constexpr int ES = T == G4_F32 ? 4 : T == G4_KV_Q8 ? 1 : 2; };

// element i of a register's worth of cached elements (16-bit and fp32 values, codes)
template <int T>
__device__ __forceinline__ float cached(const uint32_t* w, int i) {
    if constexpr (T == G4_F32) return __uint_as_float(w[i]);
    else if constexpr (T == G4_F16) return hbits_to_f32(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu);
    else if constexpr (T == G4_BF16) return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    else return (float)(int8_t)(w[i >> 2] >> (8 * (i & 3)));
}
// N elements that lie next to each other
template <int T, int N>
__device__ __forceinline__ void load_cached(const uint8_t* at, float (&x)[N]) {
    constexpr int B = N * Cached<T>::ES;
    uint32_t w[(B + 3) / 4];
    if constexpr (B >= 16) {
#pragma unroll
        for (int i = 0; i < B / 16; i++) {
            // 16 bytes are next to each other in a block, the next 16 are a token's next lane's
            const uint4 y = *reinterpret_cast<const uint4*>(at + i * 256);
            w[4 * i] = y.x; w[4 * i + 1] = y.y; w[4 * i + 2] = y.z; w[4 * i + 3] = y.w;
        }
    } else if constexpr (B == 8) {
        const uint2 y = *reinterpret_cast<const uint2*>(at);
        w[0] = y.x; w[1] = y.y;
    } else if constexpr (B == 4) {
        w[0] = *reinterpret_cast<const uint32_t*>(at);
    } else if constexpr (B == 2) {
        w[0] = *reinterpret_cast<const uint16_t*>(at);
    } else {
        w[0] = *at;
    }
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = cached<T>(w, i);
}

// One wave: one q row's head (dims lane * N .. + N - 1, times scale log2(e))
// over positions first .. last of sequence s, `step` times four at a time
// from the four that hold position at on; adds to the running maximum m, sum
// l and o.  fp32 throughout; only the positions asked for have a part, so
// that infinities and NaN elsewhere do not matter; where a page is none: NaN.
template <int TC, int HD>
__device__ void row_keys(const KvPool& p, int s, int kvh, int first, int last, int at, int step, const float (&q)[HD / 64],
                         float& m, float& l, float (&o)[HD / 64]) {
    constexpr int ES = Cached<TC>::ES, N = HD / 64;
    const int lane = threadIdx.x & 63;
    for (int t0 = at & ~3; t0 <= last; t0 += 4 * step) {
        const int page = p.page_of(s, t0);
        const size_t block = p.block_of(page < 0 ? 0 : page, kvh, t0), off = block * (16 * HD * ES);
        const uint8_t* kb = p.kp + off;
        const uint8_t* vb = p.vp + off;
        const float* ks = reinterpret_cast<const float*>(p.kp + p.scale_off) + block * 16 + (t0 & 15);
        const float* vs = reinterpret_cast<const float*>(p.vp + p.scale_off) + block * 16 + (t0 & 15);
        float x[4], v[N][4], mn = m;
#pragma unroll
        for (int i = 0; i < N; i++) load_cached<TC, 4>(vb + kv_v_byte<ES>(t0 & 15, lane * N + i), v[i]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float k[N];
            load_cached<TC, N>(kb + kv_k_byte<ES>((t0 & 15) + j, lane * N), k);
            x[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < N; i++) x[j] = __builtin_fmaf(q[i], k[i], x[j]);
            x[j] = wave_sum(x[j]);
            if (TC == G4_KV_Q8) x[j] *= ks[j];
            if (page < 0) x[j] = __uint_as_float(0x7fc00000u);
            if (t0 + j < first || t0 + j > last) x[j] = -INFINITY;
            mn = fmaxf(mn, x[j]);
        }
        const float f = exp2f(m - mn);
        l *= f;
        m = mn;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] *= f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (t0 + j < first || t0 + j > last) continue;
            const float w = exp2f(x[j] - mn);
            l += w;
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = __builtin_fmaf(w, TC == G4_KV_Q8 ? v[i][j] * vs[j] : v[i][j], o[i]);
        }
    }
}

// ---- few keys: one launch, fp32 throughout, a workgroup a row and head ------------
// Taken by what a call can ask for at most, its rows and the keys that the
// window or the table allows, in units of 512 bytes of a key's row (fewer take
// as long): up to 256 keys a row and 2^17 of all rows and heads.  8 heads, this
// against the tiles and the join: bf16 of 256, 8 rows of 64 / 128 / 256 / 512 keys
// 5.8 / 8.2 / 13.7 / 24.5 and 18.4 / 18.4 / 20.0 / 21.4 us, 64 rows of 128 / 256 keys
// 11.6 / 20.4 and 19.2 / 20.6, 512 rows of 64 keys 28.2 and 19.2; fp32 of 512, 8 rows
// of 64 / 128 keys 13.3 / 23.8 and 25.7 / 24.7, 64 rows of 64 keys 24.6 and 25.9; codes
// of 128, 128 rows of 64 / 128 / 256 keys 8.8 / 14.9 / 27.2 and 14.6 / 15.7 / 17.6.
template <int TQ, int TC, int HD>
__global__ __launch_bounds__(256) void attn_chunk_row_kernel(ChunkArgs a) {
    typedef typename RowElem<TQ>::t E;
    constexpr int N = HD / 64;
    const int row = blockIdx.x, h = blockIdx.y, kvh = h / a.group;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float red[4][HD + 2];
    const SeqAt sq = find_seq(a.cu, a.lens, a.n_seqs, 1, 0, 0, (unsigned)row);
    if (sq.r0 < 0 || sq.r1 > a.m || row < sq.r0 || row >= sq.r1 || sq.r1 - sq.r0 > sq.len || !a.p.fits(sq.len)) return;
    const int last = sq.len - sq.r1 + row, first = a.window > 0 && last >= a.window ? last + 1 - a.window : 0;
    const E* qr = (const E*)a.q + (size_t)row * a.q_stride + (size_t)h * HD + lane * N;
    float q[N], o[N] = {}, m = -FLT_MAX, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) q[i] = (float)qr[i] * (a.scale * kLog2e);
    row_keys<TC, HD>(a.p, sq.s, kvh, first, last, (first & ~3) + 4 * wave, 4, q, m, l, o);
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

// ---- second launch: items of more than one share ---------------------------------
// The first border inside an item stands for the item.  A workgroup takes every
// gridDim.x-th of all such borders' units, 32 columns and 128 dims (64 where there
// are no more), and joins the pieces with the weights 2^(m_i - max m), four at a
// time.  What bounds it: the chain flags - list - pieces (7 us for 23 rows of one
// sequence, 2 of it the launch).  A workgroup for every border and unit, of which most
// have nothing to do: 19 us where this takes 15, 40 sequences of a row and one of 471.
constexpr int kJoinWG = 1024;
template <int TQ, int HD>
__global__ __launch_bounds__(256) void attn_chunk_join_kernel(ChunkArgs a) {
    typedef typename RowElem<TQ>::t E;
    constexpr int D = HD < 128 ? HD : 128, V = D / 32, B = 4;     // dims, 16-byte values of a thread, pieces at a time
    __shared__ unsigned flags[kShares + 1];
    __shared__ int list[kShares + 1], cnt[4], ends[4], found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, h = lane >> 5;
    const Notes* notes = reinterpret_cast<const Notes*>(a.part);
    const int shares = 1 << a.lg;
    // what the threads before this one have, and all of them
    auto before = [&](int v, int& all) {
        const int x = (int)wave_scan((u64)v);
        lds_sync();
        if (lane == 63) cnt[wave] = x;
        lds_sync();
        int k = x - v;
        all = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i < wave) k += cnt[i];
            all += cnt[i];
        }
        return k;
    };
    const unsigned mine = tid < shares ? notes->flags[tid] : 0;
    flags[tid] = mine;
    if (tid == 0) flags[kShares] = 0;
    lds_sync();
    // thread t: units of the item that goes out of share t
    const int cols_out = mine & kGoesOut ? (int)(flags[tid + 1] >> kColsShift) : 0, units = (cols_out + 31) / 32 * (HD / D);
    int n;
    const int unit0 = before(units, n);
    for (int unit = blockIdx.x; unit < n; unit += gridDim.x) {
        if (unit >= unit0 && unit < unit0 + units) {
            found[0] = tid + 1;
            found[1] = unit - unit0;
        }
        lds_sync();
        const int w = found[0], slot = found[1] / (HD / D), z = found[1] % (HD / D), ncols = (int)(flags[w] >> kColsShift);
        const ShareNote to = notes->item[w];
        // the shares that the item goes through, up to the one that it ends in, and which
        // of them have tiles; in order, so that sums are the same every time
        const unsigned f = w + tid < shares ? flags[w + tid] : 0;
        const u64 stop = __ballot(!(f & kGoesThrough));
        if (lane == 0) ends[wave] = stop ? __builtin_ctzll(stop) : 64;
        lds_sync();
        int last = 0;
        for (int i = 0; i < 4; i++) {
            last += ends[i];
            if (ends[i] < 64) break;
        }
        const bool in = tid <= last && f & kTilesIn;
        const int first = flags[w - 1] & kTilesOut ? 1 : 0;
        int pieces;
        const int k = before(in ? 1 : 0, pieces) + first;
        pieces += first;
        if (in) list[k] = (w + tid) * 2 + (f & kFromTile0 ? 1 : 0);
        if (first && tid == 0) list[0] = (w - 1) * 2 + 1;
        lds_sync();
        // one piece alone has been written
        if (pieces > 1 && slot * 32 + col < ncols) {
            const size_t at = (size_t)slot * HD * 32 + (size_t)z * D * 32 + tid * 4;
            const size_t ml = (size_t)a.cols * HD + ((z * D >= 256 ? a.cols : 0) + slot * 32 + col) * 2;
            f4_t x[V] = {};
            float m = -FLT_MAX, l = 0.0f;
            for (int i = 0; i < pieces; i += B) {
                float2 y[B];
                f4_t v[B][V];
#pragma unroll
                for (int j = 0; j < B; j++) {
                    const int p = list[i + j < pieces ? i + j : i];
                    const float* from = a.part + sizeof(Notes) / 4 + (size_t)p * part_floats(a.cols, HD);
                    y[j] = *reinterpret_cast<const float2*>(from + ml);
#pragma unroll
                    for (int k = 0; k < V; k++) v[j][k] = *reinterpret_cast<const f4_t*>(from + at + k * 1024);
                }
                float top = m;
#pragma unroll
                for (int j = 0; j < B; j++) top = fmaxf(top, y[j].x);
                // (fp32 V: l may be as far above its piece's products as 2^203)
                const float f = exp2f(m - top);
                l = move_sum(l, m - top);
                m = top;
#pragma unroll
                for (int k = 0; k < V; k++) x[k] *= f;
#pragma unroll
                for (int j = 0; j < B; j++) {
                    if (i + j >= pieces) break;
                    const float f = exp2f(y[j].x - top);
                    l += move_sum(y[j].y, y[j].x - top);
#pragma unroll
                    for (int k = 0; k < V; k++)
#pragma unroll
                        for (int c = 0; c < 4; c++) x[k][c] = __builtin_fmaf(f, v[j][k][c], x[k][c]);
                }
            }
            const int c = slot * 32 + col, r = (int)((unsigned)c * ((65535u + to.nh) / (unsigned)to.nh) >> 16), hh = c - r * to.nh;
            E* out = (E*)a.out + (size_t)(to.row + r) * a.out_stride + (size_t)(to.head + hh) * HD + z * D;
            const float s = 1.0f / l;
#pragma unroll
            for (int k = 0; k < V; k++) {
                // registers 4 b .. + 3 of 32-dim tile k: dims 8 b + 4 h .. + 3, or 4 b + 2 h, 16
                // more, and one more of each
                const int b = wave;
                const E y[4] = {(E)(x[k][0] * s), (E)(x[k][1] * s), (E)(x[k][2] * s), (E)(x[k][3] * s)};
                if (a.pairs) {
                    const E y2[4] = {y[0], y[2], y[1], y[3]};
                    E* at = out + k * 32 + 4 * b + 2 * h;
                    __builtin_memcpy(__builtin_assume_aligned(at, 2 * sizeof(E)), y2, 2 * sizeof(E));
                    __builtin_memcpy(__builtin_assume_aligned(at + 16, 2 * sizeof(E)), y2 + 2, 2 * sizeof(E));
                } else {
                    __builtin_memcpy(__builtin_assume_aligned(out + k * 32 + 8 * b + 4 * h, 4 * sizeof(E)), y, 4 * sizeof(E));
                }
            }
        }
        lds_sync();   // the list is the next unit's
    }
}

// columns of a workgroup, and what follows from it
void set_columns(ChunkArgs& a, int cols) {
    a.gh = a.group < cols ? a.group : cols;
    a.ngrp = (a.group + a.gh - 1) / a.gh;
    a.rpi = cols / a.gh;
    const long used = (long)a.m * a.gh;
    a.cols = used < cols ? (int)((used + 31) / 32 * 32) : cols;
    // the most that the line can measure: fewer shares, fewer workgroups
    double keys = (double)(a.p.table_stride * (1l << a.p.lgpage));
    if (a.window > 0 && a.window < keys) keys = a.window;
    const double most = ((double)a.m / a.rpi + a.n_seqs) * (keys + a.rpi + kLead) * a.p.n_kv * a.ngrp / kLeast;
    a.lg = 0;
    while (a.lg < kLgShares && (2 << a.lg) <= most) a.lg++;
}

template <int TQ, int TC, int HD, bool SMALL>
int launch_tiles(ChunkArgs a) {
    typedef Plan<TQ, TC, HD> P;
    set_columns(a, P::COLS);
    a.pairs = P::M::kPairs;
    // (a scale of 0: rows of zeros, and a score of -infinity times fq has to stay one)
    a.fq = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
    if (SMALL) {
        int e;
        a.fq = frexpf(fabsf(a.scale), &e) * kLog2e;
        a.by = ldexpf(1.0f, e);
    }
    auto kernel = attn_chunk_kernel<TQ, TC, HD, SMALL>;
    // more than 64 KB of LDS has to be asked for, once on each device
    static std::atomic<unsigned long long> asked{0};
    int dev = 0;
    G4_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !(asked >> dev & 1)) {
        G4_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, P::LDS));
        if (dev < 64) asked |= 1ull << dev;
    }
    hipLaunchKernelGGL(kernel, dim3(1 << a.lg), dim3(64 * P::NW), P::LDS, g4_stream(), a);
    if (a.lg == 0) return g4_check_launch("attn_chunk_kernel");   // nothing to join
    const int units = ((1 << a.lg) - 1) * (a.cols / 32) * (HD < 128 ? 1 : HD / 128);
    hipLaunchKernelGGL((attn_chunk_join_kernel<TQ, HD>), dim3(units < kJoinWG ? units : kJoinWG), dim3(256), 0, g4_stream(), a);
    return g4_check_launch("attn_chunk_kernel");
}
template <int TQ, int TC, int HD>
int launch_chunk(const ChunkArgs& a) {
    double keys = (double)a.p.table_stride * (1 << a.p.lgpage);
    if (a.window > 0 && a.window < keys) keys = a.window;
    constexpr int ES = Mode<TQ, TC>::ES, kUnit = HD * ES > 512 ? HD * ES / 512 : 1;
    if (keys * kUnit <= kFewKeys && keys * kUnit * a.m * a.n_heads <= kFewPairs) {
        hipLaunchKernelGGL((attn_chunk_row_kernel<TQ, TC, HD>), dim3(a.m, a.n_heads), dim3(256), 0, g4_stream(), a);
        return g4_check_launch("attn_chunk_row_kernel");
    }
    if constexpr (TQ == G4_BF16) {
        if (a.scale != 0.0f && fabsf(a.scale) < 1.0f) return launch_tiles<TQ, TC, HD, true>(a);
    }
    return launch_tiles<TQ, TC, HD, false>(a);
}
template <int TQ, int TC>
int launch_chunk(const ChunkArgs& a, int hd) {
    if (hd == 64) return launch_chunk<TQ, TC, 64>(a);
    if (hd == 128) return launch_chunk<TQ, TC, 128>(a);
    if (hd == 256) return launch_chunk<TQ, TC, 256>(a);
    return launch_chunk<TQ, TC, 512>(a);
}

}  // namespace
}  // namespace g4

using namespace g4;

extern "C" size_t g4_attn_chunk_paged_part_bytes(int m, int n_heads, int n_kv, int hd) {
    if (m < 1 || n_heads < 1 || n_heads > 65535 || n_kv < 1 || n_heads % n_kv || (hd != 64 && hd != 128 && hd != 256 && hd != 512))
        return 0;
    // two partial results of each share
    const int group = n_heads / n_kv, cols = 128, gh = group < cols ? group : cols;
    const long used = (long)m * gh;
    return sizeof(Notes) + (size_t)kShares * 2 * part_floats(used < cols ? (int)((used + 31) / 32 * 32) : cols, hd) * 4;
}

extern "C" int g4_attn_chunk_paged(const void* q, int q_stride, int q_type, const void* kp, const void* vp, int type,
                                   int n_pages, int page, int n_kv, int hd, const int* table, int table_stride, const int* cu,
                                   const int* lens, int n_seqs, int m, int window, int n_heads, float attn_scale, void* part,
                                   void* out, int out_stride) {
    const char* who = "g4_attn_chunk_paged";
    ChunkArgs a = {};
    const int rc = kv_pool_check(who, &a.p, kp, vp, type, n_pages, page, n_kv, hd, table, table_stride);
    if (rc) return rc;
    const int es = q_type == G4_F32 ? 4 : q_type == G4_F16 || q_type == G4_BF16 ? 2 : 0;
    G4_CHECK(es && (q_type == G4_F32 || q_type == type || (q_type == G4_BF16 && type == G4_KV_Q8)), G4_ERR_TYPE,
             "%s: rows of type %d over a cache of type %d", who, q_type, type);
    G4_CHECK_ARG(n_heads > 0 && n_heads <= 65535 && n_heads % n_kv == 0 && window >= 0, "%s: %d heads over %d kv heads, window %d",
                 who, n_heads, n_kv, window);
    G4_CHECK_ARG(q && cu && lens && part && out && al16(q) && al16(part) && al16(out), "%s: null or unaligned pointer", who);
    G4_CHECK_ARG(q_stride % (16 / es) == 0 && q_stride / hd >= n_heads && out_stride % (16 / es) == 0 && out_stride / hd >= n_heads,
                 "%s: strides %d, %d (multiples of %d, n_heads * hd at least)", who, q_stride, out_stride, 16 / es);
    G4_CHECK_ARG(n_seqs > 0 && n_seqs <= kKvMaxSeqs && m > 0, "%s: %d rows of %d sequences (1 to %d)", who, m,
                 n_seqs, kKvMaxSeqs);
    a.q = q; a.out = out; a.cu = cu; a.lens = lens; a.part = (float*)part; a.q_stride = q_stride; a.out_stride = out_stride;
    a.n_seqs = n_seqs; a.m = m; a.window = window; a.n_heads = n_heads; a.scale = attn_scale;
    a.group = n_heads / n_kv;
    if (q_type == G4_F32) {
        if (type == G4_F32) return launch_chunk<G4_F32, G4_F32>(a, hd);
        if (type == G4_F16) return launch_chunk<G4_F32, G4_F16>(a, hd);
        if (type == G4_BF16) return launch_chunk<G4_F32, G4_BF16>(a, hd);
        return launch_chunk<G4_F32, G4_KV_Q8>(a, hd);
    }
    if (q_type == G4_F16) return launch_chunk<G4_F16, G4_F16>(a, hd);
    if (type == G4_BF16) return launch_chunk<G4_BF16, G4_BF16>(a, hd);
    return launch_chunk<G4_BF16, G4_KV_Q8>(a, hd);
}
