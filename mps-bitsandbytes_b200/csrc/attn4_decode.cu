// Attention over the paged 4-bit cache for few query rows per sequence (single tokens, drafts) - and, row tile by row
// tile, for any number of them.  out = softmax(scale q K^T) V, K = code * absmax, V = code * absmax.
//
// Bound: HBM, for the cached bytes (head_dim / 2 + 2 head_dim / blocksize per token, head and side) are read once and
// the arithmetic per byte is small; what stands in the way is turning 4-bit codes into operands at that rate.
//
//  * Work is a list of (sequence, kv head, row tile, 16-token key tile), cut into equal runs of tiles, one per CTA,
//    whatever the sequences' lengths are: the lengths are read on the device, so a captured graph follows them.
//    A run that begins or ends inside a (sequence, head, row tile) leaves a partial result in the workspace, and
//    attn4_combine_kernel joins the partials.
//  * A key tile is one group of the cache: one bulk copy into the warp's own ring of stages.  No barrier between warps
//    while tiles stream; a warp waits on its own mbarriers only.
//  * S^T = K Q^T and O^T = V^T P^T with mma.m16n8k16: tokens (then channels) are the 16 rows and the query rows
//    the 8 columns, so a group of up to 8 heads wastes nothing of the tile.  (tcgen05 would want 128 rows and the
//    operands in shared memory: here they are made in registers.)  Codes become fp16 pairs by a 256-entry table
//    of byte -> (low nibble's value, high nibble's), held once per lane so that 32 look-ups never meet in a bank.
//    For V the pair has to run along tokens: the nibbles of two tokens' words are first brought into one byte.
//  * A block's absmax multiplies the fp32 score (K) or the probability (V), never a code: K enters the product
//    with the rounding of the 16 code values to fp16 only.
//  * Softmax: probabilities are 2^(x - m) with a reference m that follows the running maximum only when a score
//    exceeds it by 2^8: one vote per tile instead of a reduction, and fp32 sums lose nothing by it.  The weight
//    p * absmax goes to fp16; absmax is taken times a power of two that is lowered, in the same vote, when it exceeds 2^7.
//    bf16 queries are brought to fp16 by a power of two per row: exact, but for parts below 2^-24 of the row's largest.
#include <type_traits>

#include "attn4.cuh"
#include "ops.cuh"

namespace mpsbnb {

using namespace sm100;

static __device__ int g_attn4_status = 0;

constexpr int AD_WARPS = 8;                                          // of a team: the warps that share a run of tiles
constexpr int AD_STAGES = 3;
constexpr uint32_t AD_LUT = 65536;                                   // shared-window address of the table
constexpr uint32_t AD_BASE = 1024;                                   // ... and of the dynamic shared memory

// A block has one table (256 entries of 256 bytes, the lower 128 of which are in use: lane l's copy at 4 l) on a 64 KB
// boundary, so that one byte permute makes a look-up's address.  It is too large for two blocks on an SM; instead a
// block holds TEAMS teams of eight warps which do not wait on one another.
template <int D, int BS, int NT> struct AdSmem {
    static constexpr int TEAMS = D * NT <= 128 ? 2 : 1;              // by registers (accumulators and q): 128 or 255 a thread
    static constexpr int THREADS = TEAMS * AD_WARPS * 32;
    static constexpr int GROUP = 2 * kv4_half_bytes(D, BS);
    static constexpr int RT = 8 * NT;
    static constexpr int RED_LD = 64 + 4;                            // floats per row of a merge pass
    // window addresses: half of the warps' rings before the table, the other half and the rest behind it
    static constexpr int RING_HALF = TEAMS * AD_WARPS / 2 * AD_STAGES * GROUP;
    static constexpr uint32_t RING0 = AD_BASE, RING1 = AD_LUT + 65536;
    static constexpr uint32_t RED = RING1 + RING_HALF;
    static constexpr uint32_t STAT = RED + TEAMS * AD_WARPS * RT * RED_LD * 4;   // (maximum, sum) of every warp and row
    static constexpr uint32_t BAR = STAT + TEAMS * AD_WARPS * RT * 8;
    static constexpr uint32_t END = BAR + TEAMS * AD_WARPS * AD_STAGES * 8 + 16;
    static constexpr int BYTES = END - AD_BASE;
    static_assert(RING0 + RING_HALF <= AD_LUT && BYTES <= 227 * 1024, "shared memory of the decode kernel");
    static_assert(RING_HALF % 128 == 0, "stages start on 16-byte boundaries");
};

// value pair of byte `byte` of word; lut = AD_LUT + 4 lane, whose second byte is free
__device__ __forceinline__ uint32_t ad_lut(uint32_t lut, uint32_t word, int byte) {
    uint32_t v;
    asm("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(__byte_perm(word, lut, 0x7604 | (byte << 4))));
    return v;
}
__device__ __forceinline__ void ad_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t ad_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t ad_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// NB consecutive 16-bit absmax values as floats
template <typename T, int NB> __device__ __forceinline__ void ad_scales(uint32_t addr, float (&s)[NB]) {
    uint32_t w[(NB + 1) / 2];
    if constexpr (NB == 1) { uint16_t h; asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(addr) : "memory"); w[0] = h; }
    else if constexpr (NB == 2) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr) : "memory");
    else if constexpr (NB == 4) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
    else asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        s[i] = to_f32<T>(*reinterpret_cast<const T *>(&h));
    }
}

// A walk over the pieces (runs of key tiles of one sequence, head and row tile) of a team's run of tiles.
struct AdPiece {
    Attn4Seq s;
    int b, h, r;                                 // sequence, kv head, row tile
    int a, e;                                    // key tiles of the piece, relative to s.tlo
    int64_t left;                                // tiles of the run after this piece

    // first piece of the run [t0, t1) of the whole list; whole warp
    __device__ __forceinline__ void start(const Attn4Args &A, int rt, int64_t t0, int64_t t1) {
        const int lane = threadIdx.x & 31;
        int64_t base = 0;
        for (int b0 = 0;; b0 += 32) {
            Attn4Seq q;
            int64_t w = 0;
            if (b0 + lane < A.sq.batch) { q.get(A, b0 + lane, rt); w = q.work(A.kv.kv_heads); }
            int64_t inc = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += up;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, base + inc > t0);
            if (hit != 0) {
                const int l = __ffs(hit) - 1;
                b = b0 + l;
                base += __shfl_sync(0xffffffffu, inc - w, l);
                break;
            }
            base += __shfl_sync(0xffffffffu, inc, 31);
        }
        s.get(A, b, rt);
        const int64_t off = t0 - base;
        const int sub = (int)(off / s.nt);
        h = sub / s.rts;
        r = sub - h * s.rts;
        a = (int)(off - (int64_t)sub * s.nt);
        left = t1 - t0;
        e = (int)min((int64_t)s.nt, a + left);
        left -= e - a;
    }
    // next piece; false when the run is done
    __device__ __forceinline__ bool next(const Attn4Args &A, int rt) {
        if (left == 0) return false;
        if (++r == s.rts) {
            r = 0;
            if (++h == A.kv.kv_heads) {
                h = 0;
                do { ++b; s.get(A, b, rt); } while (s.nt == 0);
            }
        }
        a = 0;
        e = (int)min((int64_t)s.nt, left);
        left -= e;
        return true;
    }
};

// tiles per team: equal, and a multiple of a team's warps
__device__ __forceinline__ int64_t ad_per(int64_t total, int teams) {
    const int64_t per = (total + teams - 1) / teams;
    return (per + AD_WARPS - 1) / AD_WARPS * AD_WARPS;
}
// partial result of team c, slot s (0: its first piece, 1: its last): RT x D sums, then RT (maximum, sum) pairs
template <int D, int RT> __device__ __forceinline__ float *ad_partial(float *ws, int64_t c, int s) {
    return ws + (c * 2 + s) * (RT * (D + 2));
}

template <int D, int BS, int NT, typename T>
__global__ void __launch_bounds__((AdSmem<D, BS, NT>::THREADS), 1)
attn4_decode_kernel(const __grid_constant__ Attn4Args A) {
    using S = AdSmem<D, BS, NT>;
    constexpr int NB = D / BS, MT = D / 16, MB = BS / 16, RT = S::RT;   // MB: k steps, and channel tiles, per block
    constexpr int HALF = kv4_half_bytes(D, BS), SOFF = KV4_GROUP * (D / 2);
    constexpr int WARPS = S::TEAMS * AD_WARPS;
    extern __shared__ __align__(128) unsigned char smem[];
    if (smem_u32(smem) != AD_BASE) {                                 // the layout counts on it
        if (threadIdx.x == 0) atomicExch(&g_attn4_status, 403);
        return;
    }
    const int cta_warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int in_team = cta_warp / AD_WARPS, warp = cta_warp % AD_WARPS;
    const int team = blockIdx.x * S::TEAMS + in_team;
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + (S::END - 16 - AD_BASE));

    // ------------------------------------------------------------ my team's run
    int64_t unused, total;
    attn4_prefix(A, RT, 0, unused, total);
    const int64_t per = ad_per(total, gridDim.x * S::TEAMS);
    const int64_t t0 = min(total, team * per), t1 = min(total, t0 + per);
    pdl_launch_dependents();
    if (blockIdx.x * S::TEAMS * per >= total) return;                // nothing for any team of the block

    // ------------------------------------------------------------ table, barriers
    {
        const float mine = kCode[A.quant_type][lane & 15] * attn4_code_scale(A.quant_type);
        for (int b = cta_warp; b < 256; b += WARPS) {
            const float lo = __shfl_sync(0xffffffffu, mine, b & 15), hi = __shfl_sync(0xffffffffu, mine, b >> 4);
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(AD_LUT + (uint32_t)(b * 256 + lane * 4)), "r"(ad_half2(lo, hi)) : "memory");
        }
        if (threadIdx.x == 0) {
            for (int i = 0; i < WARPS * AD_STAGES; ++i) mbar_init(S::BAR + 8 * i, 1);
            *abort_flag = 0;
            fence_mbar_init();
        }
    }
    __syncthreads();
    if (t0 >= t1) return;                                            // whole team; no barrier of the block follows
    auto team_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(in_team + 1), "n"(AD_WARPS * 32) : "memory"); };
    const uint32_t lut = AD_LUT + lane * 4;
    const uint32_t ring = cta_warp < WARPS / 2 ? S::RING0 + cta_warp * (AD_STAGES * S::GROUP) : S::RING1 + (cta_warp - WARPS / 2) * (AD_STAGES * S::GROUP);
    const uint32_t bars = S::BAR + cta_warp * AD_STAGES * 8;
    const bool negate = A.scale_log2 < 0.0f;                         // a negative scale goes into q: maxima stay maxima

    // ------------------------------------------------------------ producer side: this warp's tiles, in order
    AdPiece in;                                                      // piece the next copy belongs to
    in.start(A, RT, t0, t1);
    AdPiece cur = in;
    bool in_more = true;
    int in_k = 0, in_page = 0;                                       // tile ordinal within the piece; pages of 32 ordinals
    uint32_t put = 0;                                                // next stage to fill
    auto issue = [&]() {                                             // whole warp
        while (in_more) {
            const int t = in.a + warp + in_k * AD_WARPS;
            if (t < in.e && (in.s.tlo + t) * 16 < in.s.len) break;
            in_more = in.next(A, RT);
            in_k = 0;
        }
        if (!in_more) return;
        if ((in_k & 31) == 0) {
            const int t = in.a + warp + (in_k + lane) * AD_WARPS;
            in_page = -1;
            if (t < in.e) in_page = __ldg(A.sq.table + (int64_t)in.b * A.sq.table_ld + (((in.s.tlo + t) * 16) >> A.kv.page_shift));
        }
        const int page = __shfl_sync(0xffffffffu, in_page, in_k & 31);
        const int place = (in.s.tlo + in.a + warp + in_k * AD_WARPS) * 16;
        const uint32_t st = put;
        if (page >= 0 && page < A.kv.num_pages) {
            if (lane == 0) {
                mbar_arrive_expect_tx(bars + 8 * st, S::GROUP);
                bulk_load_1d(ring + st * S::GROUP, A.kv.group(page, in.h, place), S::GROUP, bars + 8 * st);
            }
        } else {
            // a page outside the cache: its keys' absmax is NaN, and so is every row that sees them
            for (int i = lane; i < KV4_GROUP * NB; i += 32)
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(ring + st * S::GROUP + SOFF + 2 * i), "h"((uint16_t)0x7fff) : "memory");
            __syncwarp();
            if (lane == 0) { atomicExch(&g_attn4_status, KV4_BAD_PAGE); mbar_arrive(bars + 8 * st); }
        }
        put = put == AD_STAGES - 1 ? 0 : put + 1;
        ++in_k;
    };
#pragma unroll 1
    for (int i = 0; i < AD_STAGES; ++i) issue();

    // ------------------------------------------------------------ consumer side
    uint32_t got = 0, phase = 0;                                     // next stage to read, its barrier's parity
    bool first_piece = true;
    do {
        const Attn4Seq &sq = cur.s;
        const int first = sq.len - sq.n;
        // q as the B operand: lane (g, c) holds row g's channels blk * BS + c * (BS / 4) + ks * 4 + 0 .. 3
        uint32_t qf[NT][NB * MB][2];
        float f[NT][2];                                              // score -> power of two, columns 2c and 2c + 1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int R = cur.r * RT + nt * 8 + g, i = R / A.group, hg = R - i * A.group;
            const bool ok = i < sq.n;
            const T *src = reinterpret_cast<const T *>(A.q) + (int64_t)(sq.row0 + i) * A.q_ts + (int64_t)(cur.h * A.group + hg) * A.q_hs;
            uint2 raw[NB * MB];
#pragma unroll
            for (int k = 0; k < NB * MB; ++k) {
                raw[k] = make_uint2(0u, 0u);
                if (ok) raw[k] = __ldg(reinterpret_cast<const uint2 *>(src + (k / MB) * BS + c * (BS / 4) + (k % MB) * 4));
                if (negate) { raw[k].x ^= 0x80008000u; raw[k].y ^= 0x80008000u; }
            }
            float fr = fabsf(A.scale_log2) * attn4_code_unscale(A.quant_type);
            if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
                uint32_t mx = 0;                                     // largest magnitude of the row, as bits of bf16
#pragma unroll
                for (int k = 0; k < NB * MB; ++k) {
                    const uint32_t x = raw[k].x & 0x7fff7fffu, y = raw[k].y & 0x7fff7fffu;
                    mx = max(max(mx, x & 0xffffu), max(x >> 16, max(y & 0xffffu, y >> 16)));
                }
                mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const int e = max(1, min(253, (int)(mx >> 7)));      // biased exponent of the largest
                const float down = __int_as_float((254 - e) << 23);  // 2^(127 - e): the largest comes to [1, 2)
                fr *= __int_as_float(e << 23);
#pragma unroll
                for (int k = 0; k < NB * MB; ++k) {
                    raw[k].x = ad_half2(__uint_as_float(raw[k].x << 16) * down, __uint_as_float(raw[k].x & 0xffff0000u) * down);
                    raw[k].y = ad_half2(__uint_as_float(raw[k].y << 16) * down, __uint_as_float(raw[k].y & 0xffff0000u) * down);
                }
            }
#pragma unroll
            for (int k = 0; k < NB * MB; ++k) { qf[nt][k][0] = raw[k].x; qf[nt][k][1] = raw[k].y; }
            fr = fmaxf(fr, 0x1p-126f);                               // scale 0: -inf * f has to stay -inf
            f[nt][0] = __shfl_sync(0xffffffffu, fr, 8 * c);          // row 2c lives in lanes (2c, *)
            f[nt][1] = __shfl_sync(0xffffffffu, fr, 8 * c + 4);
        }
        // keys that column col sees: places low[] <= place < lim[]
        int lim[NT][2], low[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int i = (cur.r * RT + nt * 8 + 2 * c + j) / A.group;
                lim[nt][j] = i < sq.n ? (A.causal ? first + i + 1 : sq.len) : 0;
                low[nt][j] = A.window > 0 ? lim[nt][j] - A.window : 0;
            }
        const int i0 = (cur.r * RT) / A.group, i1 = min(sq.n - 1, (cur.r * RT + RT - 1) / A.group);
        // places that some row sees: [any_lo, any_hi)
        const int any_lo = A.window > 0 ? first + i0 + 1 - A.window : 0, any_hi = A.causal ? first + i1 + 1 : sq.len;
        const int full_lo = A.window > 0 ? first + i1 + 1 - A.window : 0, full_hi = A.causal ? first + i0 + 1 : sq.len;

        float o[MT][NT][4], m[NT][2], l[NT][2], up = 0x1p100f;       // up: power of two that the values' absmax is taken times
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][nt][j] = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) { m[nt][j] = ATTN4_NONE; l[nt][j] = 0.0f; }

#pragma unroll 1
        for (int t = cur.a + warp; t < cur.e; t += AD_WARPS) {
            const int place0 = (sq.tlo + t) * 16;
            if (place0 >= sq.len) break;                             // the dead tile of an empty sequence
            const uint32_t st = got;
            if (!mbar_wait(bars + 8 * st, phase, abort_flag)) { atomicExch(&g_attn4_status, 402); *abort_flag = 1; }
            const uint32_t kb = ring + st * S::GROUP, vb = kb + HALF;
            // A-operand row r of the tile is token r / 2 (even r) or r / 2 + 4 (odd r), + 8 for rows 8 .. 15: the k index
            // of P^T below then gives a lane the tokens c, c + 4, c + 8, c + 12
            const int tok = (g >> 1) + 4 * (g & 1);
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[nt][j] = 0.0f;
            {
                float sc0[NB], sc1[NB];
                ad_scales<T, NB>(kb + SOFF + tok * NB * 2, sc0);
                ad_scales<T, NB>(kb + SOFF + (tok + 8) * NB * 2, sc1);
#pragma unroll
                for (int blk = 0; blk < NB; ++blk) {
                    uint32_t w0[MB / 2], w1[MB / 2];
                    const uint32_t ka = kb + tok * (D / 2) + blk * (BS / 2) + c * (BS / 8);
                    if constexpr (BS == 64) {
                        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w0[0]), "=r"(w0[1]) : "r"(ka) : "memory");
                        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w1[0]), "=r"(w1[1]) : "r"(ka + 8 * (D / 2)) : "memory");
                    } else {
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w0[0]) : "r"(ka) : "memory");
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w1[0]) : "r"(ka + 8 * (D / 2)) : "memory");
                    }
                    float acc[NT][4];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[nt][j] = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < MB; ++ks) {
                        const uint32_t x0 = w0[ks / 2], x1 = w1[ks / 2];
                        const int by = 2 * (ks & 1);
                        const uint32_t a0 = ad_lut(lut, x0, by), a1 = ad_lut(lut, x1, by), a2 = ad_lut(lut, x0, by + 1), a3 = ad_lut(lut, x1, by + 1);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) ad_mma(acc[nt], a0, a1, a2, a3, qf[nt][blk * MB + ks][0], qf[nt][blk * MB + ks][1]);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        s[nt][0] = fmaf(sc0[blk], acc[nt][0], s[nt][0]); s[nt][1] = fmaf(sc0[blk], acc[nt][1], s[nt][1]);
                        s[nt][2] = fmaf(sc1[blk], acc[nt][2], s[nt][2]); s[nt][3] = fmaf(sc1[blk], acc[nt][3], s[nt][3]);
                    }
                }
            }
            float sv0[NB], sv1[NB], sm = 0.0f;
            ad_scales<T, NB>(vb + SOFF + tok * NB * 2, sv0);
            ad_scales<T, NB>(vb + SOFF + (tok + 8) * NB * 2, sv1);
            // s[nt][0..1]: token tok, columns 2c and 2c + 1; s[nt][2..3]: token tok + 8
            const bool masked = place0 < full_lo || place0 + 16 > full_hi;   // (full_hi <= len)
            uint32_t seen = 0;                                       // bit nt * 4 + j
            if (masked) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int place = place0 + tok + 8 * (j >> 1);
                        if (place < lim[nt][j & 1] && place >= low[nt][j & 1]) seen |= 1u << (nt * 4 + j);
                        else s[nt][j] = __int_as_float(0xff800000);
                    }
                // whatever lies in a place that no row sees
                const bool in0 = place0 + tok >= any_lo && place0 + tok < any_hi, in1 = place0 + tok + 8 >= any_lo && place0 + tok + 8 < any_hi;
#pragma unroll
                for (int blk = 0; blk < NB; ++blk) { sv0[blk] = in0 ? sv0[blk] : 0.0f; sv1[blk] = in1 ? sv1[blk] : 0.0f; }
            }
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {
                sv0[blk] *= up; sv1[blk] *= up;
                sm = fmaxf(sm, fmaxf(sv0[blk], sv1[blk]));
            }
            float p[NT][4], top = -1.0f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    p[nt][j] = fmaf(s[nt][j], f[nt][j & 1], -m[nt][j & 1]);
                    top = fmaxf(top, p[nt][j]);
                }
            // p and absmax * up stay under 2^8 and 2^7, their product is at home in fp16
            if (__any_sync(0xffffffffu, top > 8.0f || sm > 128.0f)) {
                // (from the absmax itself: times `up` it may have left fp32)
                ad_scales<T, NB>(vb + SOFF + tok * NB * 2, sv0);
                ad_scales<T, NB>(vb + SOFF + (tok + 8) * NB * 2, sv1);
                const bool in0 = place0 + tok >= any_lo && place0 + tok < any_hi, in1 = place0 + tok + 8 >= any_lo && place0 + tok + 8 < any_hi;
                sm = 0.0f;
#pragma unroll
                for (int blk = 0; blk < NB; ++blk) {
                    sv0[blk] = in0 ? sv0[blk] : 0.0f; sv1[blk] = in1 ? sv1[blk] : 0.0f;
                    sm = fmaxf(sm, fmaxf(sv0[blk], sv1[blk]));
                }
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) sm = fmaxf(sm, __shfl_xor_sync(0xffffffffu, sm, d));
                float ku = 1.0f;
                if (sm * up > 128.0f) {                              // the largest comes to [16, 32)
                    const int e = max(5, (int)(__float_as_uint(fminf(sm, 3.4e38f)) >> 23));
                    const float un = __int_as_float((258 - e) << 23);   // 2^(131 - e)
                    ku = un * __frcp_rn(up);                         // (0 where the difference leaves fp32)
                    up = un;
                }
#pragma unroll
                for (int blk = 0; blk < NB; ++blk) { sv0[blk] *= up; sv1[blk] *= up; }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float mx = fmaxf(s[nt][j], s[nt][j + 2]) * f[nt][j];
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                        const float mn = mx > m[nt][j] + 8.0f ? mx : m[nt][j], k = ex2(m[nt][j] - mn);
                        m[nt][j] = mn;
                        l[nt][j] *= k;
#pragma unroll
                        for (int i = 0; i < MT; ++i) { o[i][nt][j] *= k * ku; o[i][nt][j + 2] *= k * ku; }
                        p[nt][j] = fmaf(s[nt][j], f[nt][j], -mn);
                        p[nt][j + 2] = fmaf(s[nt][j + 2], f[nt][j], -mn);
                    }
            }
            float wt[NB][NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    p[nt][j] = ex2(p[nt][j]);
                    l[nt][j & 1] += p[nt][j];
#pragma unroll
                    for (int blk = 0; blk < NB; ++blk) wt[blk][nt][j] = p[nt][j] * (j < 2 ? sv0[blk] : sv1[blk]);
                }
            if (masked) {                                            // a value that is not finite is no matter of rows that do not see it
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (!(seen >> (nt * 4 + j) & 1u)) {
#pragma unroll
                            for (int blk = 0; blk < NB; ++blk) wt[blk][nt][j] = 0.0f;
                        }
            }
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {
                uint32_t b0[NT], b1[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    b0[nt] = ad_transpose(ad_half2(wt[blk][nt][0], wt[blk][nt][1]));
                    b1[nt] = ad_transpose(ad_half2(wt[blk][nt][2], wt[blk][nt][3]));
                }
                // lane (g, c): channels blk * BS + g * (BS / 8) + 0 .. BS / 8 - 1 of the tokens c, c + 4, c + 8, c + 12
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t va = vb + (c + 4 * i) * (D / 2) + blk * (BS / 2) + g * (BS / 16);
                    if constexpr (BS == 64) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(va) : "memory");
                    else { uint16_t h; asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(va) : "memory"); w[i] = h; }
                }
                const uint32_t ev0 = (w[0] & 0x0F0F0F0Fu) | ((w[1] << 4) & 0xF0F0F0F0u), od0 = ((w[0] >> 4) & 0x0F0F0F0Fu) | (w[1] & 0xF0F0F0F0u);
                const uint32_t ev1 = (w[2] & 0x0F0F0F0Fu) | ((w[3] << 4) & 0xF0F0F0F0u), od1 = ((w[2] >> 4) & 0x0F0F0F0Fu) | (w[3] & 0xF0F0F0F0u);
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    const uint32_t a0 = ad_lut(lut, ev0, j), a1 = ad_lut(lut, od0, j), a2 = ad_lut(lut, ev1, j), a3 = ad_lut(lut, od1, j);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) ad_mma(o[blk * MB + j][nt], a0, a1, a2, a3, b0[nt], b1[nt]);
                }
            }
            if (++got == AD_STAGES) { got = 0; phase ^= 1; }
            __syncwarp();                                            // every lane has read the stage
            issue();
        }

        // ------------------------------------------------------------ join the warps
        float *red = reinterpret_cast<float *>(smem + (S::RED - AD_BASE)) + in_team * (AD_WARPS * RT * S::RED_LD);
        float2 *stat = reinterpret_cast<float2 *>(smem + (S::STAT - AD_BASE)) + in_team * (AD_WARPS * RT);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], d);
                if (g == 0) stat[warp * RT + nt * 8 + 2 * c + j] = make_float2(m[nt][j], l[nt][j]);
            }
        team_sync();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float M = m[nt][j];
#pragma unroll
                for (int w = 0; w < AD_WARPS; ++w) M = fmaxf(M, stat[w * RT + nt * 8 + 2 * c + j].x);
                const float k = ex2(m[nt][j] - M) * __frcp_rn(up) * attn4_code_unscale(A.quant_type);
#pragma unroll
                for (int i = 0; i < MT; ++i) { o[i][nt][j] *= k; o[i][nt][j + 2] *= k; }
            }
        const bool whole = cur.a == 0 && cur.e == sq.nt;
        float *part = ad_partial<D, RT>(A.ws, team, first_piece ? 0 : 1);
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += 64) {                         // 64 channels per pass
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const int mt = d0 / 16 + i4, blk = mt / MB, j2 = mt % MB;
                const int d = blk * BS + g * (BS / 8) + 2 * j2 - d0;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        *reinterpret_cast<float2 *>(red + (warp * RT + nt * 8 + 2 * c + j) * S::RED_LD + d) = make_float2(o[mt][nt][j], o[mt][nt][j + 2]);
            }
            team_sync();
            for (int x = warp * 32 + lane; x < RT * 32; x += AD_WARPS * 32) {
                const int row = x >> 5, d = 2 * (x & 31);
                const int R = cur.r * RT + row, i = R / A.group;
                if (i < sq.n) {
                    float M = stat[row].x, L = 0.0f;
                    float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int w = 1; w < AD_WARPS; ++w) M = fmaxf(M, stat[w * RT + row].x);
#pragma unroll
                    for (int w = 0; w < AD_WARPS; ++w) {
                        const float2 y = *reinterpret_cast<const float2 *>(red + (w * RT + row) * S::RED_LD + d), z = stat[w * RT + row];
                        v.x += y.x; v.y += y.y;
                        L = fmaf(z.y, ex2(z.x - M), L);
                    }
                    if (whole) {
                        const float inv = L == 0.0f ? 0.0f : __fdividef(1.0f, L);
                        const int64_t orow = (int64_t)(sq.row0 + i) * A.heads + cur.h * A.group + (R - i * A.group);
                        T pr[2] = {from_f32<T>(v.x * inv), from_f32<T>(v.y * inv)};
                        *reinterpret_cast<uint32_t *>(reinterpret_cast<T *>(A.out) + orow * D + d0 + d) = *reinterpret_cast<const uint32_t *>(pr);
                        if (A.lse != nullptr && d0 == 0 && d == 0) A.lse[orow] = L == 0.0f ? __int_as_float(0xff800000) : (M + __log2f(L)) * 0.69314718f;
                    } else {
                        *reinterpret_cast<float2 *>(part + row * D + d0 + d) = v;
                        if (d0 == 0 && d == 0) *reinterpret_cast<float2 *>(part + RT * D + 2 * row) = make_float2(M, L);
                    }
                }
            }
            team_sync();                                         // red (and, at the end, stat) may be written again
        }
        first_piece = false;
    } while (cur.next(A, RT));
}

// Joins the partial results of one (sequence, head, row tile, row): sum of 2^(m_i - M) O_i over sum of 2^(m_i - M) l_i.
template <int D, int RT, typename T>
__global__ void __launch_bounds__(256)
attn4_combine_kernel(const __grid_constant__ Attn4Args A, int teams, int rts_max) {
    __shared__ float red[8][D];
    __shared__ float reds[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int x = blockIdx.x;
    const int row = x % RT; x /= RT;
    const int r = x % rts_max; x /= rts_max;
    const int h = x % A.kv.kv_heads, b = x / A.kv.kv_heads;
    Attn4Seq s;
    s.get(A, b, RT);
    const int R = r * RT + row, i = R / A.group;
    int64_t before, total;
    attn4_prefix(A, RT, b, before, total);
    // every block waits, so that this kernel's end means the end of the one before it as well
    pdl_grid_dependency_wait();
    if (r >= s.rts || i >= s.n) return;                              // whole block
    const int64_t per = ad_per(total, teams);
    const int64_t t0 = before + (int64_t)(h * s.rts + r) * s.nt, c0 = t0 / per, c1 = (t0 + s.nt - 1) / per;
    if (c0 == c1) return;                                            // one team had it all and has written it
    float M = ATTN4_NONE;
    for (int64_t ci = c0 + lane; ci <= c1; ci += 32)
        M = fmaxf(M, ad_partial<D, RT>(A.ws, ci, t0 <= ci * per ? 0 : 1)[RT * D + 2 * row]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float L = 0.0f, v[D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) v[j] = 0.0f;
    for (int64_t ci = c0 + warp; ci <= c1; ci += 8) {
        const float *p = ad_partial<D, RT>(A.ws, ci, t0 <= ci * per ? 0 : 1);
        const float2 ml = *reinterpret_cast<const float2 *>(p + RT * D + 2 * row);
        const float k = ex2(ml.x - M);
        L = fmaf(ml.y, k, L);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) v[j] = fmaf(p[row * D + j * 32 + lane], k, v[j]);
    }
#pragma unroll
    for (int j = 0; j < D / 32; ++j) red[warp][j * 32 + lane] = v[j];
    if (lane == 0) reds[warp] = L;
    __syncthreads();
    L = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) L += reds[w];
    const float inv = L == 0.0f ? 0.0f : __fdividef(1.0f, L);
    const int64_t orow = (int64_t)(s.row0 + i) * A.heads + h * A.group + (R - i * A.group);
    for (int d = threadIdx.x; d < D; d += 256) {
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) y += red[w][d];
        reinterpret_cast<T *>(A.out)[orow * D + d] = from_f32<T>(y * inv);
    }
    if (A.lse != nullptr && threadIdx.x == 0) A.lse[orow] = L == 0.0f ? __int_as_float(0xff800000) : (M + __log2f(L)) * 0.69314718f;
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
// 16 rows per tile where 8 do not hold a sequence's rows: the keys are then expanded half as often
static int ad_nt(const mpsbnb_kv4_seqs *s, int group) { return (int64_t)s->new_tokens * group > 8 ? 2 : 1; }

static int ad_teams(int D, int NT) { return sm_count() * (D * NT <= 128 ? 2 : 1); }

template <int D, int BS, int NT, typename T>
static int ad_launch(const Attn4Args &a, int rts_max, cudaStream_t st) {
    using S = AdSmem<D, BS, NT>;
    static bool configured[64] = {};
    int dev = 0;
    MPSBNB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        MPSBNB_CUDA_TRY(cudaFuncSetAttribute(attn4_decode_kernel<D, BS, NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const int teams = ad_teams(D, NT);
    attn4_decode_kernel<D, BS, NT, T><<<teams / S::TEAMS, S::THREADS, S::BYTES, st>>>(a);
    int rc = check_launch();
    if (rc != MPSBNB_OK) return rc;
    const int64_t blocks = (int64_t)a.sq.batch * a.kv.kv_heads * rts_max * S::RT;
    if (blocks > 0x7fffffffll) return MPSBNB_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    MPSBNB_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn4_combine_kernel<D, S::RT, T>, a, teams, rts_max));
    return check_launch();
}

template <int D, int BS>
static int ad_launch_t(const Attn4Args &a, int dtype, int nt, int rts_max, cudaStream_t st) {
    if (dtype == MPSBNB_F16) return nt == 1 ? ad_launch<D, BS, 1, __half>(a, rts_max, st) : ad_launch<D, BS, 2, __half>(a, rts_max, st);
    return nt == 1 ? ad_launch<D, BS, 1, __nv_bfloat16>(a, rts_max, st) : ad_launch<D, BS, 2, __nv_bfloat16>(a, rts_max, st);
}

int attn4_decode_status_fetch(int *out, bool reset) {
    MPSBNB_CUDA_TRY(cudaMemcpyFromSymbol(out, g_attn4_status, sizeof(int)));
    if (reset) {
        const int zero = 0;
        MPSBNB_CUDA_TRY(cudaMemcpyToSymbol(g_attn4_status, &zero, sizeof(int)));
    }
    return MPSBNB_OK;
}

}  // namespace mpsbnb

using namespace mpsbnb;

extern "C" size_t mpsbnb_attention_4bit_workspace_bytes(const mpsbnb_kv4_cache *cache, const mpsbnb_kv4_seqs *seqs, int heads) {
    if (kv4_check_cache(cache, 0) != MPSBNB_OK || kv4_check_seqs(seqs, cache) != MPSBNB_OK) return 0;
    if (heads <= 0 || heads % cache->kv_heads != 0 || seqs->batch == 0 || seqs->tokens == 0) return 0;
    const int nt = ad_nt(seqs, heads / cache->kv_heads);
    return (size_t)ad_teams(cache->head_dim, nt) * 2 * (8 * nt) * (cache->head_dim + 2) * sizeof(float);
}

extern "C" int mpsbnb_attention_4bit(const mpsbnb_kv4_cache *cache, int layer, const mpsbnb_kv4_seqs *seqs, const void *q,
                                     int64_t q_token_stride, int64_t q_head_stride, int heads, int causal, int window, float scale,
                                     void *out, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = kv4_check_cache(cache, layer);
    if (rc == MPSBNB_OK) rc = kv4_check_seqs(seqs, cache);
    if (rc != MPSBNB_OK) return rc;
    if (heads <= 0 || heads % cache->kv_heads != 0 || window < 0 || (window > 0 && !causal)) return MPSBNB_ERR_INVALID_ARG;
    if (q_token_stride < 0 || q_head_stride < 0) return MPSBNB_ERR_INVALID_ARG;
    if (seqs->batch == 0 || seqs->tokens == 0 || seqs->new_tokens == 0) return MPSBNB_OK;
    if (q == nullptr || out == nullptr) return MPSBNB_ERR_INVALID_ARG;
    const int group = heads / cache->kv_heads;
    if ((int64_t)seqs->new_tokens * group > 0x3fffffffll) return MPSBNB_ERR_TOO_LARGE;
    if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < mpsbnb_attention_4bit_workspace_bytes(cache, seqs, heads)) return MPSBNB_ERR_WORKSPACE;
    // rows are fetched in 16-byte pieces
    if (!aligned16(q) || ((q_token_stride | q_head_stride) & 7) != 0 || !aligned16(out)) return MPSBNB_ERR_UNSUPPORTED;
    Attn4Args a;
    a.kv = kv4_layer(cache, layer);
    a.sq = kv4_seqs(seqs, cache);
    a.q = q; a.q_ts = q_token_stride; a.q_hs = q_head_stride;
    a.out = out; a.lse = lse; a.ws = (float *)workspace;
    a.heads = heads; a.group = group; a.causal = causal != 0; a.window = window; a.quant_type = cache->quant_type;
    a.scale_log2 = scale * 1.4426950408889634f;
    if ((int64_t)seqs->new_tokens * group >= 128) return attn4_prompt(a, cache->head_dim, cache->blocksize, cache->dtype, (cudaStream_t)stream);
    const int nt = ad_nt(seqs, group);
    const int rts_max = (seqs->new_tokens * group + 8 * nt - 1) / (8 * nt);
    cudaStream_t st = (cudaStream_t)stream;
    const int dt = cache->dtype;
    if (cache->blocksize == 32) {
        if (cache->head_dim == 64) return ad_launch_t<64, 32>(a, dt, nt, rts_max, st);
        if (cache->head_dim == 128) return ad_launch_t<128, 32>(a, dt, nt, rts_max, st);
        return ad_launch_t<256, 32>(a, dt, nt, rts_max, st);
    }
    if (cache->head_dim == 64) return ad_launch_t<64, 64>(a, dt, nt, rts_max, st);
    if (cache->head_dim == 128) return ad_launch_t<128, 64>(a, dt, nt, rts_max, st);
    return ad_launch_t<256, 64>(a, dt, nt, rts_max, st);
}
