// kv_page.hip -- the paged KV cache: rows stored into pages (rounded or
// quantised on the way) and read back as fp32 rows.
#include <math.h>

#include "g4_kvpage.h"
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

// A workgroup's share: up to 16 rows of one sequence that fall into one
// 16-token block of the cache, of one kv head, K (blockIdx.z 0) or V.
// Sequence s takes the units (cu[s] >> 4) + 2 s onwards: its n rows touch at
// most (n + 30) / 16 blocks, so the shares never overlap and no prefix sum is
// needed; units past a sequence's last block have nothing to do.
struct Unit {
    int s, at;         // sequence, position of the block's token 0
    int t0, t1;        // tokens of the block that take part
    int row;           // row of token 0 of the block (may lie before the first row)
};

__device__ __forceinline__ bool find_unit(const RowArgs& a, Unit& u) {
    const unsigned id = blockIdx.x;
    const SeqAt q = find_seq(a.cu, a.lens, a.n_seqs, 1, 4, 2, id);
    if (q.r0 < 0 || q.r1 <= q.r0 || q.r1 > a.m || q.r1 - q.r0 > q.len || !a.p.fits(q.len)) return false;
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

// Rows of 16 tokens are rounded in registers, put into the block's order in
// LDS and written as whole 16-byte pieces; where only some of a piece's tokens
// take part (K pieces belong to one token, V pieces to four) only those are
// written.
// Q8: d = max|x| / 127 and codes rint(x / d), both fp32 divisions, so that a
// code is the nearest one and what is read back is the same wherever it is
// computed; a row with an infinity or NaN gets the scale NaN.
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
    if (!find_unit(a, u)) return;
    const int page = a.p.page_of(u.s, u.at);   // on its way beside the rows
    const bool is_v = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* __restrict__ src = (is_v ? a.v : a.k) + (size_t)blockIdx.y * HD;
    const int sub = lane / M::LPR, col = lane % M::LPR;
    // whether any of a pass's rows of this wave takes part
    auto in_use = [&](int i) {
        const int t = (i * 4 + __builtin_amdgcn_readfirstlane(wave)) * M::RPW;
        return t + M::RPW > u.t0 && t < u.t1;
    };
    float4 x[M::PASS][M::VPL];
#pragma unroll
    for (int i = 0; i < M::PASS; i++) {
        const int t = (i * 4 + wave) * M::RPW + sub;
        if (!in_use(i)) continue;
        // rows that take no part read the block's first row in their place
        const int r = u.row + (t >= u.t0 && t < u.t1 ? t : u.t0);
#pragma unroll
        for (int k = 0; k < M::VPL; k++)
            x[i][k] = *reinterpret_cast<const float4*>(src + (size_t)r * a.kv_stride + (k * M::LPR + col) * 4);
    }
    if (page < 0) return;
    uint8_t* pool = is_v ? a.p.vp : a.p.kp;
    const size_t block = a.p.block_of(page, blockIdx.y, u.at);
#pragma unroll
    for (int i = 0; i < M::PASS; i++) {
        const int t = (i * 4 + wave) * M::RPW + sub;
        if (!in_use(i)) continue;
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
                reinterpret_cast<float*>(pool + a.p.scale_off)[block * 16 + t] = d;
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
    if (!find_unit(a, u)) return;
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
