// qkv_seqs.hip -- norms of q, k and v heads with the rotation at each packed
// row's own position, as rows of a type or straight into the paged KV cache.
#include <math.h>

#include "g4_kvrows.h"
#include "g4_tile.h"

namespace g4 {
namespace {

constexpr int kRun = 16;   // blocks whose workgroups are neighbours, a multiple of 8

struct PostArgs {
    KvPool p;            // pages (kp null: rows)
    const float* q;
    const float* k;
    const float* v;
    const float* q_norm;
    const float* k_norm;
    void* qo;
    void* ko;            // rows
    void* vo;
    const float2* tab;   // (cos, sin) of n_rot / 2 pairs for each position
    const int* cu;
    const int* lens;
    int q_stride, kv_stride, qo_stride, kvo_stride;
    int n_heads, n_kv, tab_rows, half, n_seqs, m;
    float eps;
};

// four elements of a row, rounded to the type
template <int RT>
__device__ __forceinline__ void store4(void* row, int c, const float4& x) {
    typedef typename Elem<RT>::t T;
    const T y[4] = {Elem<RT>::of(x.x), Elem<RT>::of(x.y), Elem<RT>::of(x.z), Elem<RT>::of(x.w)};
    __builtin_memcpy(__builtin_assume_aligned((T*)row + c, 4 * sizeof(T)), y, 4 * sizeof(T));
}

// y = x / sqrt(mean(x^2) + eps) * w, then each pair (j, j + HD / 2), j < half,
// turned by its position's angle: (a, b) -> (a cos - b sin, a sin + b cos).
// A workgroup has up to 16 rows of one block of the cache and one head: q
// heads first, then k, then v (which has neither weight nor rotation).  A row
// is in one wave (RowMap): the sum of squares is a reduction over its lanes,
// a pair's other half lies in another lane of the row or, at HD 512, in the
// lane's other four dims.  The operations and their order are those of
// g4_qkv_post_rows, so that for HD 256 and 512 the bits are.
// What bounds it: bytes, each read and written once, where there are thousands of
// rows: 8 q heads on 2 kv heads, 8191 rows of 256 into fp32 pages 34 us in a row, 3193 rows
// of 256 as bf16 14.2 us, 4.4 TB/s; 1539 rows of 512 into pages of bf16 13.8 us, 4.3.
// Up to a few dozen rows the chain cu and lens - (page,) row and angles - sum -
// store, 6 to 7 us with the launch.
// The workgroups' order: all heads of 16 blocks, then the next 16.  Workgroups go to
// the eight XCDs in turn, so an XCD has all heads of a block, one behind the other:
// it reads whole rows and finds their angles in its L2.  All blocks of a head, then
// the next head's, and this: 8191 rows into fp32 pages 46 and 34 us, 16384 96 and 85;
// bf16 of 512, 4096 rows 43 and 27, 16384 161 and 126; rows of bf16, 8191 39 and 27,
// 12000 43 and 38; but the 3193 rows 13.4 and 14.2, 1539 8.7 and 9.1.  (8, 32 and 64
// blocks: within 3 %.  Six heads a workgroup: 8191 rows 38, the 3193 21.)
// PT: type of the pages, -1: K and V as rows.  RT: type of the rows.
template <int PT, int RT, int HD>
__global__ __launch_bounds__(256) void qkv_seqs_kernel(PostArgs a) {
    typedef RowMap<HD> M;
    constexpr int ES = PT < 0 ? 1 : (int)sizeof(typename Elem<PT < 0 ? G4_F32 : PT>::t);
    __shared__ __align__(16) uint8_t img[PT < 0 ? 16 : 16 * HD * ES];
    Unit u;
    const unsigned heads = a.n_heads + 2 * a.n_kv, run = blockIdx.x / (kRun * heads), nth = blockIdx.x - run * kRun * heads;
    const unsigned unit = run * kRun + nth % kRun;
    const int b = nth / kRun;
    if (!find_unit(a.cu, a.lens, a.n_seqs, a.m, unit,
                   [&](int len) { return len <= a.tab_rows && (PT < 0 || a.p.fits(len)); }, u))
        return;
    const int kind = b < a.n_heads ? 0 : b < a.n_heads + a.n_kv ? 1 : 2;
    const int head = b - (kind == 0 ? 0 : kind == 1 ? a.n_heads : a.n_heads + a.n_kv);
    int page = 0;
    if (PT >= 0 && kind > 0) page = a.p.page_of(u.s, u.at);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int sub = lane / M::LPR, col = lane % M::LPR;
    const float* __restrict__ src = (kind == 0 ? a.q : kind == 1 ? a.k : a.v) + (size_t)head * HD;
    const int stride = kind == 0 ? a.q_stride : a.kv_stride;
    const float* __restrict__ w = kind == 0 ? a.q_norm : a.k_norm;
    float4 x[M::PASS][M::VPL], wv[M::VPL];
    float2 cs[M::PASS][4];
    // this lane's first dim and the first of its four pairs
    const bool low = M::VPL == 2 || col < M::LPR / 2;
    const int j0 = (low ? col : col - M::LPR / 2) * 4;
#pragma unroll
    for (int i = 0; i < M::PASS; i++) {
        if (!pass_in_use<HD>(u, i, wave)) continue;
        const int t = (i * 4 + wave) * M::RPW + sub, tt = t >= u.t0 && t < u.t1 ? t : u.t0;
#pragma unroll
        for (int k = 0; k < M::VPL; k++)
            x[i][k] = *reinterpret_cast<const float4*>(src + (size_t)(u.row + tt) * stride + (k * M::LPR + col) * 4);
        if (kind < 2) {
            const float2* tab = a.tab + (size_t)(u.at + tt) * a.half;
#pragma unroll
            for (int c = 0; c < 4; c++) cs[i][c] = j0 + c < a.half ? tab[j0 + c] : make_float2(1.0f, 0.0f);
        }
    }
    if (kind < 2) {
#pragma unroll
        for (int k = 0; k < M::VPL; k++) wv[k] = reinterpret_cast<const float4*>(w)[k * M::LPR + col];
    }
    if (page < 0) return;
#pragma unroll
    for (int i = 0; i < M::PASS; i++) {
        if (!pass_in_use<HD>(u, i, wave)) continue;
        float y[M::VPL][4], ss = 0.0f;
#pragma unroll
        for (int k = 0; k < M::VPL; k++) {
            y[k][0] = x[i][k].x; y[k][1] = x[i][k].y; y[k][2] = x[i][k].z; y[k][3] = x[i][k].w;
#pragma unroll
            for (int c = 0; c < 4; c++) ss += y[k][c] * y[k][c];
        }
        if (M::LPR == 64) {
            ss = wave_sum(ss);
        } else {
#pragma unroll
            for (int d = 1; d < M::LPR; d <<= 1) ss += shfl_xor(ss, d);
        }
        const float s = 1.0f / sqrtf(ss / (float)HD + a.eps);
#pragma unroll
        for (int k = 0; k < M::VPL; k++) {
            const float wk[4] = {wv[k].x, wv[k].y, wv[k].z, wv[k].w};
#pragma unroll
            for (int c = 0; c < 4; c++) y[k][c] = y[k][c] * (kind < 2 ? s * wk[c] : s);
        }
        if (kind < 2) {
            float z[M::VPL][4];
#pragma unroll
            for (int k = 0; k < M::VPL; k++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const bool first = M::VPL == 2 ? k == 0 : low;
                    const float other = M::VPL == 2 ? y[M::VPL - 1 - k][c] : shfl_xor(y[k][c], M::LPR / 2);
                    const float turned = first ? y[k][c] * cs[i][c].x - other * cs[i][c].y
                                               : other * cs[i][c].y + y[k][c] * cs[i][c].x;
                    z[k][c] = j0 + c < a.half ? turned : y[k][c];
                }
#pragma unroll
            for (int k = 0; k < M::VPL; k++)
#pragma unroll
                for (int c = 0; c < 4; c++) y[k][c] = z[k][c];
        }
#pragma unroll
        for (int k = 0; k < M::VPL; k++) x[i][k] = make_float4(y[k][0], y[k][1], y[k][2], y[k][3]);
    }
    if constexpr (PT >= 0) {
        if (kind > 0) {
            store_block<PT, HD>(a.p, page, head, u, kind == 2, x, img);
            return;
        }
    }
    typedef typename Elem<RT>::t R;
    R* dst = (R*)(kind == 0 ? a.qo : kind == 1 ? a.ko : a.vo) + (size_t)head * HD;
    const int so = kind == 0 ? a.qo_stride : a.kvo_stride;
#pragma unroll
    for (int i = 0; i < M::PASS; i++) {
        const int t = (i * 4 + wave) * M::RPW + sub;
        if (t < u.t0 || t >= u.t1) continue;
#pragma unroll
        for (int k = 0; k < M::VPL; k++) store4<RT>(dst + (size_t)(u.row + t) * so, (k * M::LPR + col) * 4, x[i][k]);
    }
}

template <int PT, int RT>
void launch_post(const PostArgs& a, int hd) {
    const dim3 grid((unsigned)(a.m / 16 + 2 * a.n_seqs + kRun - 1) / kRun * kRun * (a.n_heads + 2 * a.n_kv));
    if (hd == 64) hipLaunchKernelGGL((qkv_seqs_kernel<PT, RT, 64>), grid, dim3(256), 0, g4_stream(), a);
    else if (hd == 128) hipLaunchKernelGGL((qkv_seqs_kernel<PT, RT, 128>), grid, dim3(256), 0, g4_stream(), a);
    else if (hd == 256) hipLaunchKernelGGL((qkv_seqs_kernel<PT, RT, 256>), grid, dim3(256), 0, g4_stream(), a);
    else hipLaunchKernelGGL((qkv_seqs_kernel<PT, RT, 512>), grid, dim3(256), 0, g4_stream(), a);
}
template <int PT>
void launch_post(const PostArgs& a, int row_type, int hd) {
    if (row_type == G4_F32) launch_post<PT, G4_F32>(a, hd);
    else if (row_type == G4_F16) launch_post<PT, G4_F16>(a, hd);
    else launch_post<PT, G4_BF16>(a, hd);
}

int row_size(int type) { return type == G4_F32 ? 4 : type == G4_F16 || type == G4_BF16 ? 2 : 0; }

// what both entry points check alike: q (q or no heads), the table, the rows
int post_check(const char* who, const PostArgs& a, int hd, int n_rot, int row_type, const void* rope_tab) {
    const int unit = 16 / row_size(row_type);
    G4_CHECK_ARG(!a.q || (a.q_norm && a.qo && al16(a.q) && al16(a.q_norm) && al16(a.qo)), "%s: null or unaligned q rows", who);
    G4_CHECK_ARG(!a.q || (a.n_heads > 0 && a.n_heads <= 65535 && a.q_stride % 4 == 0 && a.q_stride / hd >= a.n_heads &&
                          a.qo_stride % unit == 0 && a.qo_stride / hd >= a.n_heads),
                 "%s: %d q heads in strides %d, %d (multiples of 4 and %d, n_heads * hd at least)", who, a.n_heads, a.q_stride,
                 a.qo_stride, unit);
    G4_CHECK_ARG((void*)a.q != a.qo || (row_type == G4_F32 && a.q_stride == a.qo_stride) || !a.q,
                 "%s: q rows in place have to be fp32 rows of one stride", who);
    G4_CHECK_ARG(rope_tab && ((uintptr_t)rope_tab & 7u) == 0 && a.tab_rows > 0 && n_rot > 0 && n_rot <= hd && n_rot % 2 == 0,
                 "%s: bad RoPE table (%d rows of %d, even and %d at most)", who, a.tab_rows, n_rot, hd);
    G4_CHECK_ARG(a.cu && a.lens && a.n_seqs > 0 && a.n_seqs <= kKvMaxSeqs && a.m > 0, "%s: %d rows of %d sequences (1 to %d)",
                 who, a.m, a.n_seqs, kKvMaxSeqs);
    G4_CHECK_ARG(kv_grid_fits(((size_t)a.m / 16 + 2 * a.n_seqs + kRun) * ((size_t)a.n_heads + 2 * a.n_kv), 256),
                 "%s: %d rows of %d heads: more than one launch takes", who, a.m, a.n_heads + 2 * a.n_kv);
    return G4_OK;
}

}  // namespace
}  // namespace g4

using namespace g4;

extern "C" int g4_qkv_post_seqs(const float* q, int q_stride, const float* q_norm, int n_heads, const float* k,
                                const float* v, int kv_stride, const float* k_norm, int n_kv, int hd, void* q_out,
                                int q_out_stride, void* k_out, void* v_out, int kv_out_stride, int type,
                                const float* rope_tab, int tab_rows, int n_rot, float eps, const int* cu, const int* lens,
                                int n_seqs, int m) {
    const char* who = "g4_qkv_post_seqs";
    G4_CHECK(row_size(type), G4_ERR_TYPE, "%s: unsupported row type %d", who, type);
    G4_CHECK_ARG(hd == 64 || hd == 128 || hd == 256 || hd == 512, "%s: head_dim %d", who, hd);
    G4_CHECK_ARG(q || k, "%s: neither q nor k", who);
    PostArgs a = {};
    a.q = q; a.q_norm = q_norm; a.qo = q_out; a.q_stride = q_stride; a.qo_stride = q_out_stride;
    a.n_heads = q ? n_heads : 0;
    a.k = k; a.v = v; a.k_norm = k_norm; a.ko = k_out; a.vo = v_out; a.kv_stride = kv_stride; a.kvo_stride = kv_out_stride;
    a.n_kv = k ? n_kv : 0;
    a.tab = (const float2*)rope_tab; a.tab_rows = tab_rows; a.half = n_rot / 2; a.eps = eps;
    a.cu = cu; a.lens = lens; a.n_seqs = n_seqs; a.m = m;
    if (k) {
        const int unit = 16 / row_size(type);
        G4_CHECK_ARG(v && k_norm && k_out && v_out && al16(k) && al16(v) && al16(k_norm) && al16(k_out) && al16(v_out),
                     "%s: null or unaligned k or v rows", who);
        G4_CHECK_ARG(n_kv > 0 && n_kv <= 32767 && kv_stride % 4 == 0 && kv_stride / hd >= n_kv && kv_out_stride % unit == 0 &&
                     kv_out_stride / hd >= n_kv,
                     "%s: %d kv heads in strides %d, %d (multiples of 4 and %d, n_kv * hd at least)", who, n_kv, kv_stride,
                     kv_out_stride, unit);
        G4_CHECK_ARG((k != k_out && v != v_out) || (type == G4_F32 && kv_stride == kv_out_stride),
                     "%s: k and v rows in place have to be fp32 rows of one stride", who);
    }
    const int rc = post_check(who, a, hd, n_rot, type, rope_tab);
    if (rc) return rc;
    launch_post<-1>(a, type, hd);
    return g4_check_launch("qkv_seqs_kernel");
}

extern "C" int g4_kv_page_append(void* kp, void* vp, int type, int n_pages, int page, int n_kv, int hd, const int* table,
                                 int table_stride, const float* k, const float* v, int kv_stride, const float* k_norm,
                                 const float* q, int q_stride, const float* q_norm, int n_heads, void* q_out,
                                 int q_out_stride, int q_type, const float* rope_tab, int tab_rows, int n_rot, float eps,
                                 const int* cu, const int* lens, int n_seqs, int m) {
    const char* who = "g4_kv_page_append";
    PostArgs a = {};
    int rc = kv_pool_check(who, &a.p, kp, vp, type, n_pages, page, n_kv, hd, table, table_stride);
    if (rc) return rc;
    G4_CHECK(!q || row_size(q_type), G4_ERR_TYPE, "%s: unsupported type %d of q rows", who, q_type);
    if (!q) q_type = G4_F32;
    G4_CHECK_ARG(k && v && k_norm && al16(k) && al16(v) && al16(k_norm), "%s: null or unaligned k or v rows", who);
    G4_CHECK_ARG(n_kv <= 32767 && kv_stride % 4 == 0 && kv_stride / hd >= n_kv,
                 "%s: %d kv heads in stride %d (a multiple of 4, n_kv * hd at least)", who, n_kv, kv_stride);
    a.q = q; a.q_norm = q_norm; a.qo = q_out; a.q_stride = q_stride; a.qo_stride = q_out_stride;
    a.n_heads = q ? n_heads : 0;
    a.k = k; a.v = v; a.k_norm = k_norm; a.kv_stride = kv_stride; a.n_kv = n_kv;
    a.tab = (const float2*)rope_tab; a.tab_rows = tab_rows; a.half = n_rot / 2; a.eps = eps;
    a.cu = cu; a.lens = lens; a.n_seqs = n_seqs; a.m = m;
    rc = post_check(who, a, hd, n_rot, q_type, rope_tab);
    if (rc) return rc;
    if (type == G4_F32) launch_post<G4_F32>(a, q_type, hd);
    else if (type == G4_F16) launch_post<G4_F16>(a, q_type, hd);
    else if (type == G4_BF16) launch_post<G4_BF16>(a, q_type, hd);
    else launch_post<G4_KV_Q8>(a, q_type, hd);
    return g4_check_launch("qkv_seqs_kernel");
}
