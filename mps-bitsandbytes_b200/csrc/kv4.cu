// The paged 4-bit key/value cache apart from its quantiser (quant4.cu) and its attention (attn4_decode.cu,
// attn4_prompt.cu): rows read back as the values they stand for, and copies of whole pages.
#include <new>

#include "kv4.cuh"

namespace mpsbnb {

static __device__ int g_kv4_status = 0;

// ------------------------------------------------------------------------------------------
// Dequantise: out[b, place, h, :] = fl(code * absmax), zeros past the sequence's end.  Bound by the 2 bytes written per
// element.  A thread owns 16 elements of K and of V (8 bytes of codes in, two 16-byte stores out each); the codebook
// sits in shared memory once per lane, so a warp's 32 look-ups never meet in a bank.
// ------------------------------------------------------------------------------------------
template <typename T, int BS>
__global__ void __launch_bounds__(256)
kv4_dequantize_kernel(const Kv4Layer kv, const Kv4Seqs sq, int quant_type, int head_dim, int max_len, T *__restrict__ k,
                      T *__restrict__ v) {
    __shared__ float tab[16 * 32];
    for (int i = threadIdx.x; i < 512; i += 256) tab[i] = kCode[quant_type][i >> 5];
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const int cpr = head_dim / 16;
    const int64_t total = (int64_t)sq.batch * max_len * kv.kv_heads * cpr;
    const int64_t stride = (int64_t)gridDim.x * 256;
    for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < total; c += stride) {
        const int64_t r = c / cpr;
        const int kc = (int)(c - r * cpr);
        const int64_t bp = r / kv.kv_heads;
        const int h = (int)(r - bp * kv.kv_heads);
        const int b = (int)(bp / max_len), place = (int)(bp - (int64_t)b * max_len);
        const int len = min(max(__ldg(sq.lens + b), 0), sq.capacity);
        uint2 kw = make_uint2(0u, 0u), vw = make_uint2(0u, 0u);
        float ks = 0.0f, vs = 0.0f;
        const bool live = place < len;
        if (live) {
            const int page = __ldg(sq.table + (int64_t)b * sq.table_ld + (place >> kv.page_shift));
            if (page < 0 || page >= kv.num_pages) {
                if (kc == 0) atomicExch(&g_kv4_status, KV4_BAD_PAGE);
                ks = vs = __int_as_float(0x7fc00000);
            } else {
                const uint8_t *g = kv.group(page, h, place);
                const int slot = place & (KV4_GROUP - 1);
                const int so = kv.scale_off + 2 * (slot * (head_dim / BS) + kc * 16 / BS);
                kw = __ldg(reinterpret_cast<const uint2 *>(g + slot * (head_dim / 2)) + kc);
                vw = __ldg(reinterpret_cast<const uint2 *>(g + kv.half_bytes + slot * (head_dim / 2)) + kc);
                ks = to_f32<T>(*reinterpret_cast<const T *>(g + so));
                vs = to_f32<T>(*reinterpret_cast<const T *>(g + kv.half_bytes + so));
            }
        }
        auto put = [&](T *out, uint2 w, float s) {
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t word = j < 4 ? w.x : w.y;
                const float lo = tab[((word >> (8 * (j & 3))) & 15u) * 32 + lane], hi = tab[((word >> (8 * (j & 3) + 4)) & 15u) * 32 + lane];
                T pr[2] = {from_f32<T>(live ? __fmul_rn(lo, s) : 0.0f), from_f32<T>(live ? __fmul_rn(hi, s) : 0.0f)};
                o[j] = *reinterpret_cast<const uint32_t *>(pr);
            }
            uint4 *dst = reinterpret_cast<uint4 *>(out + r * head_dim + kc * 16);
            __stcs(dst, make_uint4(o[0], o[1], o[2], o[3]));
            __stcs(dst + 1, make_uint4(o[4], o[5], o[6], o[7]));
        };
        put(k, kw, ks);
        put(v, vw, vs);
    }
}

// ------------------------------------------------------------------------------------------
// Page copies.  A page of a layer is one run of bytes (a multiple of 64); the pairs travel as a kernel argument, so no
// table has to be copied to the device or kept alive.  Bound by HBM: each byte once in, once out.
// ------------------------------------------------------------------------------------------
template <int N> struct PagePairs { int32_t src[N], dst[N]; };
constexpr int COPY_CHUNK = 256 * 16 * 4;                 // bytes a block moves at a time: four 16-byte loads per thread

template <int N>
__global__ void __launch_bounds__(256)
kv4_copy_kernel(uint8_t *data, int64_t layer_bytes, int64_t page_bytes, int layers, int n, const __grid_constant__ PagePairs<N> pairs) {
    const int chunks = (int)((page_bytes + COPY_CHUNK - 1) / COPY_CHUNK);
    const int64_t total = (int64_t)layers * n * chunks;
    for (int64_t i = blockIdx.x; i < total; i += gridDim.x) {
        const int64_t lp = i / chunks;
        const int ch = (int)(i - lp * chunks);
        const int l = (int)(lp / n), p = (int)(lp - (int64_t)l * n);
        const uint8_t *src = data + l * layer_bytes + pairs.src[p] * page_bytes + (int64_t)ch * COPY_CHUNK;
        uint8_t *dst = data + l * layer_bytes + pairs.dst[p] * page_bytes + (int64_t)ch * COPY_CHUNK;
        const int64_t left = page_bytes - (int64_t)ch * COPY_CHUNK;
        uint4 r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int o = (j * 256 + threadIdx.x) * 16;
            if (o < left) r[j] = __ldcs(reinterpret_cast<const uint4 *>(src + o));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int o = (j * 256 + threadIdx.x) * 16;
            if (o < left) __stcs(reinterpret_cast<uint4 *>(dst + o), r[j]);
        }
    }
}

template <int N>
static int copy_launch(const mpsbnb_kv4_cache *c, int64_t page_bytes, const int32_t *src, const int32_t *dst, int n, cudaStream_t st) {
    PagePairs<N> pairs;
    for (int i = 0; i < N; ++i) { pairs.src[i] = i < n ? src[i] : 0; pairs.dst[i] = i < n ? dst[i] : 0; }
    const int64_t total = (int64_t)c->num_layers * n * ((page_bytes + COPY_CHUNK - 1) / COPY_CHUNK);
    const int64_t cap = (int64_t)sm_count() * 8;
    kv4_copy_kernel<N><<<(int)(total < cap ? total : cap), 256, 0, st>>>((uint8_t *)c->data, c->num_pages * page_bytes, page_bytes,
                                                                       c->num_layers, n, pairs);
    return check_launch();
}

int kv4_status_fetch(int *out, bool reset) {
    MPSBNB_CUDA_TRY(cudaMemcpyFromSymbol(out, g_kv4_status, sizeof(int)));
    if (reset) {
        const int zero = 0;
        MPSBNB_CUDA_TRY(cudaMemcpyToSymbol(g_kv4_status, &zero, sizeof(int)));
    }
    return MPSBNB_OK;
}

}  // namespace mpsbnb

using namespace mpsbnb;

extern "C" size_t mpsbnb_kv4_group_bytes(int head_dim, int blocksize) {
    if (head_dim <= 0 || blocksize <= 0) return 0;
    return (size_t)(2 * kv4_half_bytes(head_dim, blocksize));
}

extern "C" size_t mpsbnb_kv4_cache_bytes(const mpsbnb_kv4_cache *c) {
    if (c == nullptr || c->num_layers <= 0 || c->num_pages <= 0 || c->kv_heads <= 0 || c->page_size <= 0 || c->head_dim <= 0 || c->blocksize <= 0) return 0;
    return (size_t)c->num_layers * (size_t)c->num_pages * (size_t)c->kv_heads * (size_t)(c->page_size / KV4_GROUP) *
           mpsbnb_kv4_group_bytes(c->head_dim, c->blocksize);
}

extern "C" int mpsbnb_kv4_dequantize(const mpsbnb_kv4_cache *cache, int layer, const mpsbnb_kv4_seqs *seqs, int64_t max_len,
                                     void *k, void *v, void *stream) {
    int rc = kv4_check_cache(cache, layer);
    if (rc != MPSBNB_OK) return rc;
    if (seqs == nullptr) return MPSBNB_ERR_INVALID_ARG;
    mpsbnb_kv4_seqs s = *seqs;
    s.cu_seqlens = nullptr; s.tokens = 0; s.new_tokens = 0;
    rc = kv4_check_seqs(&s, cache);
    if (rc != MPSBNB_OK) return rc;
    if (max_len < 0) return MPSBNB_ERR_INVALID_ARG;
    if (max_len > (1ll << 30)) return MPSBNB_ERR_TOO_LARGE;
    if (max_len == 0 || s.batch == 0) return MPSBNB_OK;
    if (k == nullptr || v == nullptr || !aligned16(k) || !aligned16(v)) return MPSBNB_ERR_INVALID_ARG;
    const Kv4Layer kv = kv4_layer(cache, layer);
    const Kv4Seqs sq = kv4_seqs(&s, cache);
    const int64_t total = (int64_t)s.batch * max_len * cache->kv_heads * (cache->head_dim / 16);
    const int64_t want = (total + 255) / 256, cap = (int64_t)sm_count() * 16;
    const int grid = (int)(want < cap ? want : cap);
    cudaStream_t st = (cudaStream_t)stream;
#define LAUNCH_DEQUANT(T, BS) \
    kv4_dequantize_kernel<T, BS><<<grid, 256, 0, st>>>(kv, sq, cache->quant_type, cache->head_dim, (int)max_len, (T *)k, (T *)v)
    if (cache->dtype == MPSBNB_F16) { if (cache->blocksize == 32) LAUNCH_DEQUANT(__half, 32); else LAUNCH_DEQUANT(__half, 64); }
    else { if (cache->blocksize == 32) LAUNCH_DEQUANT(__nv_bfloat16, 32); else LAUNCH_DEQUANT(__nv_bfloat16, 64); }
#undef LAUNCH_DEQUANT
    return check_launch();
}

extern "C" int mpsbnb_kv4_copy_pages(const mpsbnb_kv4_cache *cache, const int32_t *src, const int32_t *dst, int64_t n, void *stream) {
    int rc = kv4_check_cache(cache, 0);
    if (rc != MPSBNB_OK) return rc;
    if (n < 0 || n > cache->num_pages) return MPSBNB_ERR_INVALID_ARG;
    if (n == 0) return MPSBNB_OK;
    if (src == nullptr || dst == nullptr) return MPSBNB_ERR_INVALID_ARG;
    // the pages are moved in no particular order, so a page may not be written twice, nor read and written
    const int64_t words = (cache->num_pages + 31) / 32;
    uint32_t small[64], *seen = words <= 64 ? small : new (std::nothrow) uint32_t[words];
    if (seen == nullptr) return MPSBNB_ERR_TOO_LARGE;
    for (int64_t i = 0; i < words; ++i) seen[i] = 0;
    bool ok = true;
    for (int64_t i = 0; i < n && ok; ++i) {
        ok = dst[i] >= 0 && dst[i] < cache->num_pages && src[i] >= 0 && src[i] < cache->num_pages &&
             (seen[dst[i] >> 5] & (1u << (dst[i] & 31))) == 0;
        if (ok) seen[dst[i] >> 5] |= 1u << (dst[i] & 31);
    }
    for (int64_t i = 0; i < n && ok; ++i) ok = (seen[src[i] >> 5] & (1u << (src[i] & 31))) == 0;
    if (seen != small) delete[] seen;
    if (!ok) return MPSBNB_ERR_INVALID_ARG;
    const int64_t page_bytes = kv4_layer(cache, 0).page_bytes;
    constexpr int FEW = 32, MANY = 480;                   // 256 bytes of arguments, or just under the classic 4 KB
    for (int64_t i = 0; i < n;) {
        const int64_t left = n - i;
        const int m = (int)(left < MANY ? left : MANY);
        rc = m <= FEW ? copy_launch<FEW>(cache, page_bytes, src + i, dst + i, m, (cudaStream_t)stream)
                      : copy_launch<MANY>(cache, page_bytes, src + i, dst + i, m, (cudaStream_t)stream);
        if (rc != MPSBNB_OK) return rc;
        i += m;
    }
    return MPSBNB_OK;
}
