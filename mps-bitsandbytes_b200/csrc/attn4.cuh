// What the attention kernels over the paged 4-bit cache share: arguments, how work is laid out, how parts are joined.
#pragma once
#include "kv4.cuh"
#include "sm100.cuh"

namespace mpsbnb {

struct Attn4Args {
    Kv4Layer kv;
    Kv4Seqs sq;
    const void *q;
    int64_t q_ts, q_hs;
    void *out;
    float *lse;
    float *ws;                                   // partial results
    int32_t heads, group;                        // group: query heads per key/value head
    int32_t causal, window;
    int32_t quant_type;
    float scale_log2;                            // scale * log2(e): scores are kept as powers of two
};

// The tables hold the codebook times a constant that is divided out again in fp32.  An fp16 table of NF4 itself is off by
// 7.3e-5 in the root mean square over the codes of normal data (block maxima of 64) and by -1.1e-5 on average, and
// an average that does not vanish is not averaged away over thousands of keys; among the multiples by 1 + i 2^-22 this
// one's rounding errors are the smallest: 3.4e-5 and -1.7e-6 (of 1).  FP4's values are exact as they are.
#define ATTN4_NF4_SCALE 0x1.933fb8p+0f
__device__ __forceinline__ float attn4_code_scale(int quant_type) { return quant_type == MPSBNB_NF4 ? ATTN4_NF4_SCALE : 1.0f; }
__device__ __forceinline__ float attn4_code_unscale(int quant_type) { return quant_type == MPSBNB_NF4 ? 1.0f / ATTN4_NF4_SCALE : 1.0f; }

constexpr float ATTN4_NONE = -1e30f;             // running maximum before any key has been seen

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One sequence as the kernels walk it: rows = (new token, head of the group) pairs in tiles of `rt` rows, keys in tiles
// of 16 places.
struct Attn4Seq {
    int row0, n, len;                            // first row of q, new tokens, places
    int tlo, nt;                                 // first key tile and number of key tiles (one dead tile if there is no key)
    int rts;                                     // row tiles

    __device__ __forceinline__ void get(const Attn4Args &a, int b, int rt) {
        a.sq.get(b, row0, n, len);
        const int first = len - n;
        const int low = a.window > 0 ? max(0, first - a.window + 1) : 0;
        tlo = low >> 4;
        nt = n > 0 ? max(((len + 15) >> 4) - tlo, 1) : 0;
        rts = (n * a.group + rt - 1) / rt;
    }
    __device__ __forceinline__ int64_t work(int kv_heads) const { return (int64_t)nt * rts * kv_heads; }
};

// Tiles of all sequences before sequence b (exclusive) and of all; whole warp, same result in every lane.
__device__ __forceinline__ void attn4_prefix(const Attn4Args &a, int rt, int b, int64_t &before, int64_t &total) {
    const int lane = threadIdx.x & 31;
    int64_t bef = 0, tot = 0;
    for (int i = lane; i < a.sq.batch; i += 32) {
        Attn4Seq s;
        s.get(a, i, rt);
        const int64_t w = s.work(a.kv.kv_heads);
        tot += w;
        if (i < b) bef += w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        bef += __shfl_xor_sync(0xffffffffu, bef, o);
        tot += __shfl_xor_sync(0xffffffffu, tot, o);
    }
    before = bef;
    total = tot;
}

int attn4_prompt(const Attn4Args &a, int head_dim, int blocksize, int dtype, cudaStream_t st);   // attn4_prompt.cu

}  // namespace mpsbnb
