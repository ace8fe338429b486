// attn_chunk.hip -- attention of chunks of new rows of every sequence over the
// paged KV cache, which holds their own keys and values already.
#include "g4_attn_tile.h"
#include "g4_kvpage.h"

namespace g4 {
namespace {

struct ChunkArgs {
    KvPool p;
    const void* q;
    void* out;
    const int* cu;
    const int* lens;
    float* part;
    int q_stride, out_stride, n_seqs, m, window, n_heads;
    int group;      // q heads a kv head
    float scale;
};

template <int T>
struct Row;   // element of q and output rows
template <>
struct Row<G4_F32> { typedef float t; };
template <>
struct Row<G4_F16> { typedef _Float16 t; };
template <>
struct Row<G4_BF16> { typedef __bf16 t; };
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

// ---- one launch, fp32 throughout: a workgroup a row and head ------------------
template <int TQ, int TC, int HD>
__global__ __launch_bounds__(256) void attn_chunk_row_kernel(ChunkArgs a) {
    typedef typename Row<TQ>::t E;
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

template <int TQ, int TC, int HD>
int launch_chunk(const ChunkArgs& a) {
    hipLaunchKernelGGL((attn_chunk_row_kernel<TQ, TC, HD>), dim3(a.m, a.n_heads), dim3(256), 0, g4_stream(), a);
    return g4_check_launch("attn_chunk_row_kernel");
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
    return 16;
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
    G4_CHECK_ARG(n_seqs > 0 && n_seqs <= kKvMaxSeqs && m > 0 && kv_grid_fits(m, 256), "%s: %d rows of %d sequences (1 to %d)", who, m,
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
