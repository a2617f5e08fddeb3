// The paged 4-bit key/value cache apart from its quantiser (quant4.cu) and its attention (attn4_decode.cu,
// attn4_prompt.cu): rows read back as the values they stand for, and copies of whole pages.
#include <new>

#include "kv4.cuh"

namespace mpsbnb {

static __device__ int g_kv4_status = 0;

template <typename T> __device__ __forceinline__ uint32_t pair_of(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pair_of<__half>(float lo, float hi) { const __half2 h = __floats2half2_rn(lo, hi); return *reinterpret_cast<const uint32_t *>(&h); }
template <> __device__ __forceinline__ uint32_t pair_of<__nv_bfloat16>(float lo, float hi) { const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<const uint32_t *>(&h); }

// ------------------------------------------------------------------------------------------
// Dequantise: out[b, place, h, :] = fl(code * absmax), zeros past the sequence's end.  Bound by the 2 bytes written per
// element.  A warp takes a place, finds its page once and goes through the rows of all heads, K first; a lane owns 8 elements
// (4 bytes of codes in, a 16-byte store out), so that a warp writes 512 consecutive bytes.  The codebook sits in shared memory
// once per lane: a warp's 32 look-ups never meet in a bank.  28 900 tokens of 8 heads of 128: 38 us for 150 MB, 3.9 TB/s, 65 % of the
// issue slots.  It was 59 with half the loads under way and each place looked for only when the one before was done.
// ------------------------------------------------------------------------------------------
// two values of a word: the codes of nibbles 2 j and 2 j + 1 times s; lane: the table's address (a multiple of 2048) + 4 lane
template <typename T> __device__ __forceinline__ uint32_t kv4_pair(uint32_t w, int j, uint32_t lane, float s) {
    const uint32_t lo_at = j == 0 ? w << 7 : w >> (8 * j - 7), hi_at = j == 0 ? w << 3 : w >> (8 * j - 3);
    float lo, hi;
    asm("ld.shared.f32 %0, [%1];" : "=f"(lo) : "r"((lo_at & 0x780u) | lane));
    asm("ld.shared.f32 %0, [%1];" : "=f"(hi) : "r"((hi_at & 0x780u) | lane));
    return pair_of<T>(__fmul_rn(lo, s), __fmul_rn(hi, s));
}

template <typename T, int BS>
__global__ void __launch_bounds__(256)
kv4_dequantize_kernel(const Kv4Layer kv, const Kv4Seqs sq, int quant_type, int cpr_shift, int max_len, T *__restrict__ k,
                      T *__restrict__ v) {
    __shared__ float room[2 * 16 * 32];                  // the table, 2 KB, on a 2 KB boundary of the window somewhere in here
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(room), tab = (at + 2047u) & ~2047u;
    for (int i = threadIdx.x; i < 512; i += 256) room[(tab - at) / 4 + i] = kCode[quant_type][i >> 5];
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const uint32_t tab_lane = kv4_after_barrier(tab + lane * 4u);
    // a row is cpr chunks of 8 elements (8, 16 or 32 lanes); the warp goes on by `step` heads: 256 elements
    const int cpr = 1 << cpr_shift, step = 32 >> cpr_shift, kc = lane & (cpr - 1), rl = lane >> cpr_shift;
    const int64_t head_bytes = (int64_t)(1 << (kv.page_shift - 4)) * kv.group_bytes;
    const int64_t places = (int64_t)sq.batch * max_len;
    constexpr int U = 4;
    const int64_t warps = (int64_t)gridDim.x * 8;
    // where a place lies: its sequence's page, -1: outside the cache, -2: past the sequence's end
    auto find = [&](int64_t bp, int &place) {
        const int b = (int)(bp < 0x7fffffff ? (uint32_t)bp / (uint32_t)max_len : bp / max_len);
        place = (int)(bp - (int64_t)b * max_len);
        if (place >= min(max(__ldg(sq.lens + b), 0), sq.capacity)) return -2;
        const int page = __ldg(sq.table + (int64_t)b * sq.table_ld + (place >> kv.page_shift));
        if (page >= 0 && page < kv.num_pages) return page;
        if (lane == 0) atomicExch(&g_kv4_status, KV4_BAD_PAGE);
        return -1;
    };
    int64_t bp = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    int place = 0, page = bp < places ? find(bp, place) : -2;
    while (bp < places) {
        const int slot = place & (KV4_GROUP - 1);
        const uint8_t *src = kv.group(max(page, 0), 0, place) + rl * head_bytes + slot * (cpr * 4) + kc * 4;   // my codes of my first head's K
        const int to_scale = kv.scale_off + 2 * ((slot * cpr + kc) * 8 / BS) - (slot * (cpr * 4) + kc * 4);      // from them to their absmax
        const int64_t out = ((bp * kv.kv_heads + rl) << cpr_shift) + kc;                                       // in chunks of 8
        uint4 *dst[2] = {reinterpret_cast<uint4 *>(k) + out, reinterpret_cast<uint4 *>(v) + out};
        const bool read = page >= 0;
        const float fill = page == -1 ? __int_as_float(0x7fc00000) : 0.0f;
        const int64_t next = bp + warps;
        int next_place = 0, next_page = -2;
#pragma unroll 1
        for (int left = kv.kv_heads - rl, first = 1; left > -rl; left -= step * U, first = 0) {
            // (heads of the warp's first lanes from here on: left + rl; of mine: left)
            uint32_t w[2][U];
            float s[2][U];
#pragma unroll
            for (int side = 0; side < 2; ++side)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    w[side][u] = 0x77777777u; s[side][u] = fill;   // (code 7 is not negative: zeros, not -0)
                    if (read && u * step < left) {
                        const uint8_t *g = src + u * (step * head_bytes) + (side ? kv.half_bytes : 0);
                        w[side][u] = __ldg(reinterpret_cast<const uint32_t *>(g));
                        s[side][u] = to_f32<T>(*reinterpret_cast<const T *>(g + to_scale));
                    }
                }
            if (first && next < places) next_page = find(next, next_place);   // on its way while the codes are
#pragma unroll
            for (int side = 0; side < 2; ++side)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (u * step < left)
                        __stcs(dst[side] + 32 * u, make_uint4(kv4_pair<T>(w[side][u], 0, tab_lane, s[side][u]), kv4_pair<T>(w[side][u], 1, tab_lane, s[side][u]),
                                                              kv4_pair<T>(w[side][u], 2, tab_lane, s[side][u]), kv4_pair<T>(w[side][u], 3, tab_lane, s[side][u])));
            src += step * U * head_bytes;
            dst[0] += 32 * U; dst[1] += 32 * U;
        }
        bp = next; place = next_place; page = next_page;
    }
}

// ------------------------------------------------------------------------------------------
// Page copies.  A page of a layer is one run of bytes (a multiple of 64); the pairs travel as a kernel argument, so no
// table has to be copied to the device or kept alive.  Bound by HBM: each byte once in, once out.  666 MB of pages moved: 231 us,
// 5.8 TB/s, 0.88 of what a plain copy reaches.
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
    const int cpr_shift = cache->head_dim == 64 ? 3 : cache->head_dim == 128 ? 4 : 5;
    const int64_t want = ((int64_t)s.batch * max_len + 7) / 8, cap = (int64_t)sm_count() * 8;
    const int grid = (int)(want < cap ? want : cap);
    cudaStream_t st = (cudaStream_t)stream;
#define LAUNCH_DEQUANT(T, BS) \
    kv4_dequantize_kernel<T, BS><<<grid, 256, 0, st>>>(kv, sq, cache->quant_type, cpr_shift, (int)max_len, (T *)k, (T *)v)
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
