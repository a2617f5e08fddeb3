// What the attention kernels over the paged 4-bit cache share.
#pragma once
#include "kv4.cuh"
#include "ops.cuh"
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
    uint32_t *wide;                              // [SMs], bit b % 32: sequence b's magnitudes are too far apart for the prompt kernel
    int32_t wide_n, redo;                        // redo: those sequences and no others
    int32_t heads, group;                        // group: query heads per key/value head
    int32_t causal, window;
    int32_t quant_type;
    int32_t rows_lo, rows_hi;                    // the kernel's sequences: those of more than rows_lo and up to rows_hi rows a head
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

// Sums of probability * value are joined times this: 2^16 values of the type's largest under weights of up to 2^8 stay finite.
constexpr float ATTN4_SUM = 0x1p-24f;
constexpr float ATTN4_NONE = -0x1p127f;          // running maximum before any key has been seen
// From this reference on, the fused score * factor - reference is no longer the difference of two rounded products: for scores of 1e10
// it leaves up to 2^9 of the reference's rounding, where the largest must leave 0.
constexpr float ATTN4_FAR = 0x1p20f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Runs of work end inside a (sequence, kv head, tile of RT rows): what a run (a team's or a block's) then leaves in the workspace.
// Partial result of run c, slot s (0: its first piece, 1: its last): RT x D sums times ATTN4_SUM, then RT (reference, sum) pairs
template <int D, int RT> __device__ __forceinline__ float *attn4_partial(float *ws, int64_t c, int s) {
    return ws + (c * 2 + s) * (RT * (D + 2));
}
// behind the partials: what the run's last piece wants joined, if more runs share its (sequence, head, row tile)
struct Attn4Join {
    int n, slot;                                 // parts, in the runs from this one on (0: nothing to join); the first's slot
    int row0, rows, r, h;                        // the sequence's first row and number of (token, head) rows; row tile, kv head
};
template <int D, int RT> __device__ __forceinline__ Attn4Join *attn4_join(float *ws, int runs) {
    return reinterpret_cast<Attn4Join *>(ws + (int64_t)runs * 2 * RT * (D + 2));
}

// Joins partial results: sum of 2^(m_i - M) O_i over sum of 2^(m_i - M) l_i.  Bound by the partials' bytes and by its launch: 444
// runs of single tokens (8 rows of 128, 4 MB) 4 us behind the other kernel, 148 of prompts (256 rows, 39 MB) 14.  A block takes ROWS rows of what one run began and
// others went on with: one, whose parts its warps share, each with a running reference of its own (single tokens: up to hundreds
// of parts), or one for each warp (prompts: many rows, few parts).
constexpr int ATTN4_JOIN_WARPS = 4;
template <int D, int RT, int ROWS, typename T>
__global__ void __launch_bounds__(ATTN4_JOIN_WARPS * 32)
attn4_combine_kernel(const __grid_constant__ Attn4Args A, int runs) {
    static_assert(ROWS == 1 || ROWS == ATTN4_JOIN_WARPS, "a row for the block or for each warp");
    __shared__ float red[ATTN4_JOIN_WARPS][D + 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c0 = blockIdx.x, row = blockIdx.y * ROWS + (ROWS == 1 ? 0 : warp);
    // every block waits, so that this kernel's end means the end of the one before it as well
    sm100::pdl_grid_dependency_wait();
    const Attn4Join p = attn4_join<D, RT>(A.ws, runs)[c0];
    const int R = p.r * RT + row;
    if (p.n == 0 || R >= p.rows) return;                             // (ROWS > 1: no barrier follows)
    float M = ATTN4_NONE, L = 0.0f, v[D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) v[j] = 0.0f;
#pragma unroll 4
    for (int x = ROWS == 1 ? warp : 0; x < min(p.n, runs - c0); x += ROWS == 1 ? ATTN4_JOIN_WARPS : 1) {
        const float *q = attn4_partial<D, RT>(A.ws, c0 + x, x == 0 ? p.slot : 0);
        const float2 ml = *reinterpret_cast<const float2 *>(q + RT * D + 2 * row);
        const float mn = fmaxf(M, ml.x), ko = ex2(M - mn), kn = ex2(ml.x - mn);
        M = mn;
        L = L * ko + ml.y * kn;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) v[j] = v[j] * ko + q[row * D + j * 32 + lane] * kn;
    }
    const int i = R / A.group;
    const int64_t orow = (int64_t)(p.row0 + i) * A.heads + p.h * A.group + (R - i * A.group);
    T *const out = reinterpret_cast<T *>(A.out) + orow * D;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int j = 0; j < D / 32; ++j) red[warp][j * 32 + lane] = v[j];
        if (lane == 0) { red[warp][D] = M; red[warp][D + 1] = L; }
        __syncthreads();
        M = red[0][D];
#pragma unroll
        for (int w = 1; w < ATTN4_JOIN_WARPS; ++w) M = fmaxf(M, red[w][D]);
        float k[ATTN4_JOIN_WARPS];
        L = 0.0f;
#pragma unroll
        for (int w = 0; w < ATTN4_JOIN_WARPS; ++w) { k[w] = ex2(red[w][D] - M); L = fmaf(red[w][D + 1], k[w], L); }
        const float inv = L == 0.0f ? 0.0f : __fdividef(1.0f / ATTN4_SUM, L);
        for (int d = threadIdx.x; d < D; d += ATTN4_JOIN_WARPS * 32) {
            float y = 0.0f;
#pragma unroll
            for (int w = 0; w < ATTN4_JOIN_WARPS; ++w) y = fmaf(red[w][d], k[w], y);
            out[d] = from_f32<T>(y * inv);
        }
    } else {
        const float inv = L == 0.0f ? 0.0f : __fdividef(1.0f / ATTN4_SUM, L);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) out[j * 32 + lane] = from_f32<T>(v[j] * inv);
    }
    if (A.lse != nullptr && (ROWS == 1 ? threadIdx.x : lane) == 0) A.lse[orow] = L == 0.0f ? __int_as_float(0xff800000) : (M + __log2f(L)) * 0.69314718f;
}

// its launch behind the kernel that left the partial results
template <int D, int RT, int ROWS, typename T> static int attn4_combine(const Attn4Args &a, int runs, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(runs, RT / ROWS);
    cfg.blockDim = dim3(ATTN4_JOIN_WARPS * 32);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    MPSBNB_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn4_combine_kernel<D, RT, ROWS, T>, a, runs));
    return check_launch();
}

// Dynamic shared memory of a kernel without any other begins behind what the system keeps for itself, here at `address`?
inline bool attn4_smem_at(int dev, int address) {
    int kept = -1;
    return cudaDeviceGetAttribute(&kept, cudaDevAttrReservedSharedMemoryPerBlock, dev) == cudaSuccess && kept == address;
}

// attn4_prompt.cu; MPSBNB_ERR_UNSUPPORTED, and nothing launched, where the compiler or the device does not meet what the kernel counts on.
// split: its blocks share out the keys evenly and leave partial results.  grid: how many wrote their word of `wide`
int attn4_prompt(const Attn4Args &a, int head_dim, int blocksize, int dtype, bool split, cudaStream_t st, int *grid);
size_t attn4_prompt_ws(int head_dim);            // bytes of workspace when split

}  // namespace mpsbnb
