// attn_packed.hip -- causal attention of whole prompts, packed one after the
// other.
#include <math.h>

#include "g4_kvpage.h"
#include "g4_tile.h"

namespace g4 {
namespace {

struct PackedArgs {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    void* work;
    const int* cu;
    int q_stride, kv_stride, out_stride, n_seqs, m, window, n_heads, n_kv;
    float scale;
};

template <typename T>
__device__ __forceinline__ float to_f32(T x) { return (float)x; }

// One workgroup a row and head, a key a wave at a time.
template <typename T, int HD>
__global__ __launch_bounds__(256) void attn_packed_simple_kernel(PackedArgs a) {
    constexpr int N = HD / 64;
    const int row = blockIdx.x, h = blockIdx.y, kvh = h / (a.n_heads / a.n_kv);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float red[4][HD + 2];
    const int s = unit_seq(a.cu, a.n_seqs, 0, 0, (unsigned)row);
    const int r0 = a.cu[s], r1 = a.cu[s + 1];
    if (r0 < 0 || r1 > a.m || row < r0 || row >= r1) return;
    const int first = a.window > 0 && row - r0 >= a.window ? row + 1 - a.window : r0;
    const T* K = (const T*)a.k + (size_t)kvh * HD;
    const T* V = (const T*)a.v + (size_t)kvh * HD;
    float q[N], o[N] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++)
        q[i] = to_f32(((const T*)a.q)[(size_t)row * a.q_stride + h * HD + i * 64 + lane]) * a.scale;
    for (int t = first + wave; t <= row; t += 4) {
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) x = fmaf(q[i], to_f32(K[(size_t)t * a.kv_stride + i * 64 + lane]), x);
        x = wave_sum(x);
        const float mn = fmaxf(m, x), f = m == mn ? 1.0f : expf(m - mn), w = expf(x - mn);
        l = l * f + w;
        m = mn;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = fmaf(w, to_f32(V[(size_t)t * a.kv_stride + i * 64 + lane]), o[i] * f);
    }
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
        ((T*)a.out)[(size_t)row * a.out_stride + h * HD + d] = (T)(num / den);
    }
}

template <typename T>
void launch_packed(const PackedArgs& a, int hd) {
    const dim3 grid(a.m, a.n_heads);
    if (hd == 64) hipLaunchKernelGGL((attn_packed_simple_kernel<T, 64>), grid, dim3(256), 0, g4_stream(), a);
    else if (hd == 128) hipLaunchKernelGGL((attn_packed_simple_kernel<T, 128>), grid, dim3(256), 0, g4_stream(), a);
    else if (hd == 256) hipLaunchKernelGGL((attn_packed_simple_kernel<T, 256>), grid, dim3(256), 0, g4_stream(), a);
    else hipLaunchKernelGGL((attn_packed_simple_kernel<T, 512>), grid, dim3(256), 0, g4_stream(), a);
}

int packed_size(int type) { return type == G4_F32 ? 4 : type == G4_F16 || type == G4_BF16 ? 2 : 0; }

}  // namespace
}  // namespace g4

using namespace g4;

extern "C" size_t g4_attn_prompt_packed_work_bytes(int type, int n_seqs, int m, int n_kv, int hd) {
    if (!packed_size(type) || n_seqs < 1 || n_seqs > kKvMaxSeqs || m < 1 || n_kv < 1 || n_kv > 65535 ||
        (hd != 64 && hd != 128 && hd != 256 && hd != 512))
        return 0;
    const size_t blocks = (size_t)(m / 32 + n_seqs) * n_kv;
    return blocks * (64 * hd * (type == G4_F32 ? 4 : 2) + 32 * 8 + 16);
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
    a.q = q; a.k = k; a.v = v; a.out = out; a.work = work; a.cu = cu; a.q_stride = q_stride; a.kv_stride = kv_stride;
    a.out_stride = out_stride; a.n_seqs = n_seqs; a.m = m; a.window = window; a.n_heads = n_heads; a.n_kv = n_kv;
    a.scale = attn_scale;
    if (type == G4_F32) launch_packed<float>(a, hd);
    else if (type == G4_F16) launch_packed<_Float16>(a, hd);
    else launch_packed<__bf16>(a, hd);
    return g4_check_launch("attn_packed_kernel");
}
