// What the attention kernels over the paged 4-bit cache share.
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
    float code[16];                              // the codebook times attn4_code_scale()
};

// The tables hold the codebook times a constant that is divided out again in fp32.  An fp16 table of NF4 itself is off by
// 7.3e-5 in the root mean square over the codes of normal data (block maxima of 64) and by -1.1e-5 on average, and
// an average that does not vanish is not averaged away over thousands of keys; among the multiples by 1 + i 2^-22 this
// one's rounding errors are the smallest: 3.4e-5 and -1.7e-6 (of 1).  FP4's values are exact as they are.
#define ATTN4_NF4_SCALE 0x1.933fb8p+0f
__host__ __device__ inline float attn4_code_scale(int quant_type) { return quant_type == MPSBNB_NF4 ? ATTN4_NF4_SCALE : 1.0f; }
__device__ __forceinline__ float attn4_code_unscale(int quant_type) { return quant_type == MPSBNB_NF4 ? 1.0f / ATTN4_NF4_SCALE : 1.0f; }

constexpr float ATTN4_NONE = -1e30f;             // running maximum before any key has been seen

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

int attn4_prompt(const Attn4Args &a, int head_dim, int blocksize, int dtype, cudaStream_t st);   // attn4_prompt.cu

}  // namespace mpsbnb
