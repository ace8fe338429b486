// kv_page.hip -- the paged KV cache: rows stored into pages (rounded or
// quantised on the way) and read back as fp32 rows.
#include <math.h>

#include "g4_kvrows.h"
#include "g4_tile.h"

namespace g4 {

int kv_pool_check(const char* who, KvPool* o, const void* kp, const void* vp, int type, int n_pages, int page, int n_kv,
                  int hd, const int* table, int table_stride) {
    const size_t bytes = g4_kv_pool_bytes(type, n_pages, page, n_kv, hd);
    G4_CHECK(kv_elem_size(type), G4_ERR_TYPE, "%s: unsupported cache type %d", who, type);
    G4_CHECK_ARG(bytes, "%s: bad pool (%d pages of %d tokens, %d kv heads of %d)", who, n_pages, page, n_kv, hd);
    G4_CHECK_ARG(kp && vp && table && al16(kp) && al16(vp), "%s: null or unaligned pool", who);
    // positions and sums over 64 sequences stay within 32 bits
    G4_CHECK_ARG(table_stride > 0 && (long)table_stride * page <= 1 << 30, "%s: table_stride %d (2^30 positions at most)", who,
                 table_stride);
    o->kp = (uint8_t*)kp;
    o->vp = (uint8_t*)vp;
    o->table = table;
    o->table_stride = table_stride;
    o->n_pages = n_pages;
    o->lgpage = __builtin_ctz((unsigned)page);
    o->n_kv = n_kv;
    o->scale_off = (size_t)n_pages * page * n_kv * hd;
    return G4_OK;
}

namespace {

struct RowArgs {
    KvPool p;
    float* k;        // store: read; load: written
    float* v;
    const int* cu;
    const int* lens;
    int kv_stride, n_seqs, m;
};

// Rows rounded into pages (store_block).
// Bound by bytes: 377000 tokens of 2 x 512 in codes 0.92 ms, 4.2 TB/s read and
// written; 5136 of 2 x 256 in bf16 7.9 us with the launch, in fp32 9.1 (4.6 TB/s);
// one token each of 48 sequences 4.5 us, a chain of three round trips (rows and
// lengths, page, stores).
template <int TYPE, int HD>
__global__ __launch_bounds__(256) void kv_store_kernel(RowArgs a) {
    typedef typename Elem<TYPE>::t T;
    constexpr int ES = sizeof(T);
    typedef RowMap<HD> M;
    __shared__ __align__(16) uint8_t img[16 * HD * ES];
    Unit u;
    if (!find_unit(a.cu, a.lens, a.n_seqs, a.m, blockIdx.x, [&](int len) { return a.p.fits(len); }, u)) return;
    const int page = a.p.page_of(u.s, u.at);   // on its way beside the rows
    const bool is_v = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* __restrict__ src = (is_v ? a.v : a.k) + (size_t)blockIdx.y * HD;
    const int sub = lane / M::LPR, col = lane % M::LPR;
    float4 x[M::PASS][M::VPL];
#pragma unroll
    for (int i = 0; i < M::PASS; i++) {
        const int t = (i * 4 + wave) * M::RPW + sub;
        if (!pass_in_use<HD>(u, i, wave)) continue;
        // rows that take no part read the block's first row in their place
        const int r = u.row + (t >= u.t0 && t < u.t1 ? t : u.t0);
#pragma unroll
        for (int k = 0; k < M::VPL; k++)
            x[i][k] = *reinterpret_cast<const float4*>(src + (size_t)r * a.kv_stride + (k * M::LPR + col) * 4);
    }
    if (page < 0) return;
    store_block<TYPE, HD>(a.p, page, blockIdx.y, u, is_v, x, img);
}

// The way back: the block in 16-byte pieces into LDS, from there rows.  13098
// tokens of 2 x 256, fp16: 15.6 us, 5.2 TB/s read and written (a copy: 5.0-5.9);
// fp32 25.9, 4.1.
template <int TYPE, int HD>
__global__ __launch_bounds__(256) void kv_load_kernel(RowArgs a) {
    typedef typename Elem<TYPE>::t T;
    constexpr int ES = sizeof(T);
    typedef RowMap<HD> M;
    __shared__ __align__(16) uint8_t img[16 * HD * ES];
    Unit u;
    if (!find_unit(a.cu, a.lens, a.n_seqs, a.m, blockIdx.x, [&](int len) { return a.p.fits(len); }, u)) return;
    const bool is_v = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float* __restrict__ dst = (is_v ? a.v : a.k) + (size_t)blockIdx.y * HD;
    const uint8_t* pool = is_v ? a.p.vp : a.p.kp;
    const int page = a.p.page_of(u.s, u.at);
    const size_t block = a.p.block_of(page < 0 ? 0 : page, blockIdx.y, u.at);
    const uint8_t* in = pool + block * (16 * HD * ES);
    for (int x0 = tid; x0 < HD * ES; x0 += 256)
        reinterpret_cast<uint4*>(img)[x0] = reinterpret_cast<const uint4*>(in)[x0];
    const int sub = lane / M::LPR, col = lane % M::LPR;
    float d[M::PASS];
#pragma unroll
    for (int i = 0; i < M::PASS; i++) {
        const int t = (i * 4 + wave) * M::RPW + sub;
        d[i] = TYPE == G4_KV_Q8 ? reinterpret_cast<const float*>(pool + a.p.scale_off)[block * 16 + t] : 1.0f;
        if (page < 0) d[i] = __uint_as_float(0x7fc00000u);   // rows of a page that is none: NaN
    }
    lds_sync();
#pragma unroll
    for (int i = 0; i < M::PASS; i++) {
        const int t = (i * 4 + wave) * M::RPW + sub;
        if (t < u.t0 || t >= u.t1) continue;
#pragma unroll
        for (int k = 0; k < M::VPL; k++) {
            const int c = (k * M::LPR + col) * 4;
            float e[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const T q = *reinterpret_cast<const T*>(img + (is_v ? kv_v_byte<ES>(t, c + j) : kv_k_byte<ES>(t, c + j)));
                e[j] = Elem<TYPE>::back(q);
                if (TYPE == G4_KV_Q8) e[j] *= d[i];
                if (page < 0) e[j] = d[i];
            }
            *reinterpret_cast<float4*>(dst + (size_t)(u.row + t) * a.kv_stride + c) = make_float4(e[0], e[1], e[2], e[3]);
        }
    }
}

template <int TYPE, int HD>
void launch_rows(const RowArgs& a, bool store) {
    const dim3 grid((unsigned)(a.m / 16 + 2 * a.n_seqs), a.p.n_kv, 2);
    if (store)
        hipLaunchKernelGGL((kv_store_kernel<TYPE, HD>), grid, dim3(256), 0, g4_stream(), a);
    else
        hipLaunchKernelGGL((kv_load_kernel<TYPE, HD>), grid, dim3(256), 0, g4_stream(), a);
}
template <int TYPE>
void launch_rows(const RowArgs& a, int hd, bool store) {
    if (hd == 64) launch_rows<TYPE, 64>(a, store);
    else if (hd == 128) launch_rows<TYPE, 128>(a, store);
    else if (hd == 256) launch_rows<TYPE, 256>(a, store);
    else launch_rows<TYPE, 512>(a, store);
}

int page_rows(const char* who, RowArgs& a, const void* kp, const void* vp, int type, int n_pages, int page, int n_kv,
              int hd, const int* table, int table_stride, bool store) {
    const int rc = kv_pool_check(who, &a.p, kp, vp, type, n_pages, page, n_kv, hd, table, table_stride);
    if (rc) return rc;
    G4_CHECK_ARG(a.k && a.v && a.cu && a.lens && al16(a.k) && al16(a.v), "%s: null or unaligned rows", who);
    G4_CHECK_ARG(a.kv_stride >= 0 && a.kv_stride % 4 == 0 && a.kv_stride / hd >= n_kv,
                 "%s: kv_stride %d (a multiple of 4, n_kv * hd at least)", who, a.kv_stride);
    G4_CHECK_ARG(a.n_seqs > 0 && a.n_seqs <= kKvMaxSeqs && a.m > 0, "%s: %d rows of %d sequences (1 to %d)", who, a.m,
                 a.n_seqs, kKvMaxSeqs);
    G4_CHECK_ARG(kv_grid_fits((size_t)a.m / 16 + 2 * a.n_seqs, 256), "%s: %d rows: more than one launch takes", who, a.m);
    if (type == G4_F32) launch_rows<G4_F32>(a, hd, store);
    else if (type == G4_F16) launch_rows<G4_F16>(a, hd, store);
    else if (type == G4_BF16) launch_rows<G4_BF16>(a, hd, store);
    else launch_rows<G4_KV_Q8>(a, hd, store);
    return g4_check_launch(store ? "kv_store_kernel" : "kv_load_kernel");
}

}  // namespace
}  // namespace g4

using namespace g4;

extern "C" size_t g4_kv_pool_bytes(int type, int n_pages, int page, int n_kv, int hd) {
    const int es = kv_elem_size(type);
    if (!es || n_pages < 1 || page < 16 || page > kKvMaxPage || (page & (page - 1)) || n_kv < 1 || n_kv > 65535 ||
        (hd != 64 && hd != 128 && hd != 256 && hd != 512))
        return 0;
    const size_t rows = (size_t)n_pages * page * n_kv;   // below 2^59
    if (rows > (SIZE_MAX >> 1) / ((size_t)hd * es + 4)) return 0;
    return rows * hd * es + (type == G4_KV_Q8 ? rows * 4 : 0);
}

extern "C" int g4_kv_page_store(void* kp, void* vp, int type, int n_pages, int page, int n_kv, int hd, const int* table,
                                int table_stride, const float* k, const float* v, int kv_stride, const int* cu,
                                const int* lens, int n_seqs, int m) {
    RowArgs a = {};
    a.k = (float*)k; a.v = (float*)v; a.cu = cu; a.lens = lens; a.kv_stride = kv_stride; a.n_seqs = n_seqs; a.m = m;
    return page_rows("g4_kv_page_store", a, kp, vp, type, n_pages, page, n_kv, hd, table, table_stride, true);
}

extern "C" int g4_kv_page_load(const void* kp, const void* vp, int type, int n_pages, int page, int n_kv, int hd,
                               const int* table, int table_stride, float* k, float* v, int kv_stride, const int* cu,
                               const int* lens, int n_seqs, int m) {
    RowArgs a = {};
    a.k = k; a.v = v; a.cu = cu; a.lens = lens; a.kv_stride = kv_stride; a.n_seqs = n_seqs; a.m = m;
    return page_rows("g4_kv_page_load", a, kp, vp, type, n_pages, page, n_kv, hd, table, table_stride, false);
}
