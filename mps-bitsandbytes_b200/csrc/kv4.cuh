// Geometry of the paged 4-bit key/value cache and of a call's sequences, shared by the kernels that write it
// (quant4.cu, kv4.cu) and read it (kv4.cu, attn4_decode.cu, attn4_prompt.cu).
#pragma once
#include "common.cuh"

namespace mpsbnb {

constexpr int KV4_GROUP = 16;                    // tokens per group: the unit a kernel fetches
constexpr int KV4_BAD_PAGE = 401;                // device status: a page number outside the cache
constexpr int KV4_NO_ROOM = 430;                 // ... a new token's place behind what the page table can hold

// 16 tokens of one head: K codes, K absmax, V codes, V absmax
__host__ __device__ constexpr int kv4_half_bytes(int head_dim, int blocksize) {
    return KV4_GROUP * (head_dim / 2 + 2 * (head_dim / blocksize));
}

// One layer of the cache.
struct Kv4Layer {
    uint8_t *base;
    int64_t page_bytes;                          // kv_heads * page_size / 16 groups
    int32_t num_pages, kv_heads;
    int32_t group_bytes, page_shift;             // page_shift: log2(page_size)
    int32_t half_bytes, scale_off;               // V part of a group; absmax within a half

    // the group of 16 tokens that place pos of head h falls into, page being its (checked) page number
    __device__ __forceinline__ uint8_t *group(int page, int h, int pos) const {
        const int gpp = 1 << (page_shift - 4);
        return base + (int64_t)page * page_bytes + (int64_t)(h * gpp + ((pos >> 4) & (gpp - 1))) * group_bytes;
    }
};

struct Kv4Seqs {
    const int32_t *table, *lens, *cu;
    int64_t table_ld;
    int32_t capacity;                            // places that a row of the page table can hold
    int32_t batch, new_tokens, tokens;           // new_tokens: of every sequence where cu is null, else not looked at

    // first row of the call's tensors, number of new tokens and length of sequence b
    __device__ __forceinline__ void get(int b, int &row, int &n, int &len) const {
        if (cu != nullptr) {
            const int a = min(max(__ldg(cu + b), 0), tokens), e = min(max(__ldg(cu + b + 1), a), tokens);
            row = a;
            n = e - a;
        } else {
            row = b * new_tokens;
            n = new_tokens;
        }
        len = min(max(__ldg(lens + b), 0), capacity);
    }
    // the largest number of new tokens of a sequence; whole warp
    __device__ __forceinline__ int longest() const {
        if (cu == nullptr) return new_tokens;
        int most = 0;
        for (int b = threadIdx.x & 31; b < batch; b += 32) {
            int row, n, len;
            get(b, row, n, len);
            most = max(most, n);
        }
        return __reduce_max_sync(0xffffffffu, most);
    }
};

// A table's address that is known behind the barrier only: look-ups by it, which tell the compiler of no memory, stay there.
__device__ __forceinline__ uint32_t kv4_after_barrier(uint32_t address) {
    uint32_t same;
    asm volatile("mov.b32 %0, %1;" : "=r"(same) : "r"(address) : "memory");
    return same;
}

inline int kv4_check_cache(const mpsbnb_kv4_cache *c, int layer) {
    if (c == nullptr || c->data == nullptr || !aligned16(c->data)) return MPSBNB_ERR_INVALID_ARG;
    if (layer < 0 || layer >= c->num_layers || c->num_pages <= 0 || c->kv_heads <= 0) return MPSBNB_ERR_INVALID_ARG;
    if (!is_16bit(c->dtype) || (c->quant_type != MPSBNB_NF4 && c->quant_type != MPSBNB_FP4)) return MPSBNB_ERR_INVALID_ARG;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return MPSBNB_ERR_UNSUPPORTED;
    if (c->blocksize != 32 && c->blocksize != 64) return MPSBNB_ERR_UNSUPPORTED;
    if (!is_pow2(c->page_size) || c->page_size < 16 || c->page_size > 1024) return MPSBNB_ERR_UNSUPPORTED;
    if (c->num_pages > 0x7fffffffll || c->kv_heads > 65535) return MPSBNB_ERR_TOO_LARGE;
    return MPSBNB_OK;
}

inline Kv4Layer kv4_layer(const mpsbnb_kv4_cache *c, int layer) {
    Kv4Layer l;
    l.half_bytes = kv4_half_bytes(c->head_dim, c->blocksize);
    l.group_bytes = 2 * l.half_bytes;
    l.scale_off = KV4_GROUP * (c->head_dim / 2);
    l.page_shift = 0;
    while ((1 << l.page_shift) < c->page_size) ++l.page_shift;
    l.page_bytes = (int64_t)c->kv_heads * (c->page_size / KV4_GROUP) * l.group_bytes;
    l.num_pages = (int32_t)c->num_pages;
    l.kv_heads = c->kv_heads;
    l.base = reinterpret_cast<uint8_t *>(c->data) + (int64_t)layer * c->num_pages * l.page_bytes;
    return l;
}

inline int kv4_check_seqs(const mpsbnb_kv4_seqs *s, const mpsbnb_kv4_cache *c) {
    if (s == nullptr || s->batch < 0 || s->tokens < 0 || s->new_tokens < 0 || s->table_width < 0) return MPSBNB_ERR_INVALID_ARG;
    if (s->batch == 0) return MPSBNB_OK;
    if (s->seq_lens == nullptr || (s->table_width > 0 && (s->page_table == nullptr || s->table_ld < s->table_width))) return MPSBNB_ERR_INVALID_ARG;
    if (s->cu_seqlens == nullptr && (int64_t)s->batch * s->new_tokens != s->tokens) return MPSBNB_ERR_INVALID_ARG;
    // places and rows are 32-bit numbers in the kernels, with room for a step beyond the last
    if ((int64_t)s->table_width * c->page_size > (1ll << 30) || s->tokens > (1ll << 30)) return MPSBNB_ERR_TOO_LARGE;
    return MPSBNB_OK;
}

inline Kv4Seqs kv4_seqs(const mpsbnb_kv4_seqs *s, const mpsbnb_kv4_cache *c) {
    Kv4Seqs r;
    r.table = s->page_table; r.lens = s->seq_lens; r.cu = s->cu_seqlens; r.table_ld = s->table_ld;
    r.capacity = s->table_width * c->page_size;
    r.batch = s->batch; r.new_tokens = s->new_tokens; r.tokens = (int32_t)s->tokens;
    return r;
}

int kv4_status_fetch(int *out, bool reset);              // kv4.cu
int kv4_append_status_fetch(int *out, bool reset);       // quant4.cu
int attn4_decode_status_fetch(int *out, bool reset);     // attn4_decode.cu
int attn4_prompt_status_fetch(int *out, bool reset);     // attn4_prompt.cu

}  // namespace mpsbnb
