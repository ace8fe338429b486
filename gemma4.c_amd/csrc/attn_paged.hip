// attn_paged.hip -- attention of one new token of every sequence over the
// paged KV cache.
#include <math.h>

#include "g4_kvpage.h"
#include "g4_tile.h"

namespace g4 {
namespace {

struct PagedArgs {
    KvPool p;
    const float* q;
    float* out;
    const int* lens;
    float* part;
    int q_stride, out_stride, n_seqs, window, n_heads;
    float scale;
};

template <int TYPE>
__device__ __forceinline__ float elem(const uint8_t* p) {
    if (TYPE == G4_F32) return *reinterpret_cast<const float*>(p);
    if (TYPE == G4_F16) return (float)*reinterpret_cast<const _Float16*>(p);
    if (TYPE == G4_BF16) return bf16_to_f32(*reinterpret_cast<const uint16_t*>(p));
    return (float)*reinterpret_cast<const int8_t*>(p);
}

// One workgroup a head and sequence, a key a wave at a time:
// s_t = scale q . K_t, o = sum_t softmax(s)_t V_t with a running maximum.
template <int TYPE, int HD>
__global__ __launch_bounds__(256) void attn_paged_simple_kernel(PagedArgs a) {
    constexpr int ES = TYPE == G4_F32 ? 4 : TYPE == G4_KV_Q8 ? 1 : 2, N = HD / 64;
    const int h = blockIdx.x, s = blockIdx.y, kvh = h / (a.n_heads / a.p.n_kv);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float red[4][HD + 2];
    const int len = a.lens[s];
    bool bad = !a.p.fits(len);
    const int last = bad ? 0 : len, first = a.window > 0 && last > a.window ? last - a.window : 0;
    float q[N], o[N] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) q[i] = a.q[(size_t)s * a.q_stride + h * HD + i * 64 + lane] * a.scale;
    for (int t = first + wave; t < last; t += 4) {
        const int page = a.p.page_of(s, t);
        if (page < 0) { bad = true; break; }
        const size_t block = a.p.block_of(page, kvh, t);
        const uint8_t* kb = a.p.kp + block * (16 * HD * ES);
        const uint8_t* vb = a.p.vp + block * (16 * HD * ES);
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) x = fmaf(q[i], elem<TYPE>(kb + kv_k_byte<ES>(t & 15, i * 64 + lane)), x);
        x = wave_sum(x);
        float dv = 1.0f;
        if (TYPE == G4_KV_Q8) {
            x *= reinterpret_cast<const float*>(a.p.kp + a.p.scale_off)[block * 16 + (t & 15)];
            dv = reinterpret_cast<const float*>(a.p.vp + a.p.scale_off)[block * 16 + (t & 15)];
        }
        const float mn = fmaxf(m, x), f = m == mn ? 1.0f : expf(m - mn), w = expf(x - mn);
        l = l * f + w;
        m = mn;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = fmaf(w * dv, elem<TYPE>(vb + kv_v_byte<ES>(t & 15, i * 64 + lane)), o[i] * f);
    }
    if (bad) l = __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int i = 0; i < N; i++) red[wave][i * 64 + lane] = o[i];
    if (lane == 0) { red[wave][HD] = m; red[wave][HD + 1] = l; }
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < 4; w++) top = fmaxf(top, red[w][HD]);
    for (int d = threadIdx.x; d < HD; d += 256) {
        float num = 0.0f, den = 0.0f;
        for (int w = 0; w < 4; w++) {
            const float f = red[w][HD] == top ? 1.0f : expf(red[w][HD] - top);
            num += f * red[w][d];
            den += f * red[w][HD + 1];
        }
        a.out[(size_t)s * a.out_stride + h * HD + d] = den == 0.0f ? 0.0f : num / den;
    }
}

template <int TYPE, int HD>
void launch_paged(const PagedArgs& a) {
    hipLaunchKernelGGL((attn_paged_simple_kernel<TYPE, HD>), dim3(a.n_heads, a.n_seqs), dim3(256), 0, g4_stream(), a);
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

constexpr int kPagedWG = 512;

extern "C" size_t g4_attn_decode_paged_part_bytes(int n_heads, int n_kv, int hd) {
    if (n_heads < 1 || n_kv < 1 || n_heads % n_kv || (hd != 64 && hd != 128 && hd != 256 && hd != 512)) return 0;
    const int g = n_heads / n_kv < 16 ? n_heads / n_kv : 16;
    return (size_t)kPagedWG * 2 * g * (hd + 2) * 4;
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
    if (type == G4_F32) launch_paged<G4_F32>(a, hd);
    else if (type == G4_F16) launch_paged<G4_F16>(a, hd);
    else if (type == G4_BF16) launch_paged<G4_BF16>(a, hd);
    else launch_paged<G4_KV_Q8>(a, hd);
    return g4_check_launch("attn_paged_kernel");
}
