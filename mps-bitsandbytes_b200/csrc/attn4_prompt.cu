// Attention over the paged 4-bit cache for many query rows per sequence (prompts): out = softmax(scale q K^T) V on the
// 5th-generation tensor cores, K and V expanded from their codes into operand tiles in shared memory.
//
// Bound: the tensor pipe (4 rows keys head_dim operations) and, close behind, the exponentials (16 a clock and SM).
//
// One CTA takes 256 rows (or the last 128) of one (sequence, kv head); a row is a (new token, head of the group) pair,
// so all heads of a group share each expanded tile.  Two 128-row tiles A and B alternate: while the softmax warps of
// one work, the tensor core does the other's products.  head_dim 256 takes one tile of 128 rows (tensor memory: 256
// columns of O) and 64 keys at a time.  Roles:
//   warps 0-3, 4-7  softmax of tile A / B, one row per thread: S from tensor memory twice (maximum; exponentials), P back
//                   over S as fp16, the row's sum in fp32.  O stays in tensor memory; it is rescaled by these warps only
//                   when a row's maximum has grown by more than 2^8 since the reference was last moved.
//   warps 8-15      expand a tile of KT keys: byte -> fp16 pair by a table held once per lane, times the block's absmax,
//                   into 128-byte-swizzled panels [KT][64 channels].  For K that is the K-major operand of S = Q K^T,
//                   for V - the same layout read the other way - the MN-major operand of O = P V.
//   warp 16         issues the MMAs: S_A, S_B, then per key tile O_A += P_A V, S_A(next), O_B += P_B V, S_B(next).
//   warp 17         fetches the codes: one bulk copy per group of 16 tokens, two tiles ahead.
// fp16 operands hold bf16 caches too: the absmax of a K tile (and, carried along, of the V tiles) is brought near 2^8 by
// a power of two that the scores' factor (and the end of the row, or a rescale of O) takes back.
#include <type_traits>

#include "attn4.cuh"
#include "ops.cuh"

namespace mpsbnb {

using namespace sm100;

static __device__ int g_attn4_prompt_status = 0;

// P is 2^(x - m + 7): at most 2^15 while the reference m lags by 2^8, and what lies 2^21 below the reference still has
// fp16's full precision.
constexpr float AP_LIFT = 7.0f;
constexpr int AP_EXPAND = 8;                                         // first expander warp (of eight)
constexpr int AP_MMA = 16, AP_LOAD = 17, AP_THREADS = 18 * 32;

template <int D, int BS> struct ApSmem {
    static constexpr int TILES = D > 128 ? 1 : 2;                    // 128-row tiles
    static constexpr int KT = D > 128 ? 64 : 128;                    // keys per tile
    static constexpr int PANELS = D / 64, PANEL = KT * 128, Q_PANEL = 128 * 128;
    static constexpr int GROUP = 2 * kv4_half_bytes(D, BS), CODES = KT / KV4_GROUP * GROUP;
    static constexpr int Q = 0;
    static constexpr int K = Q + TILES * PANELS * Q_PANEL;
    static constexpr int V = K + PANELS * PANEL;
    static constexpr int LUT = V + PANELS * PANEL;
    static constexpr int RAW = LUT + 256 * 128;
    static constexpr int BAR = RAW + 2 * CODES;
    static constexpr int TOTAL = BAR + 32 * 8;
    // tensor memory columns
    static constexpr int S_COL = 0, O_COL = TILES * 128;
    static_assert(O_COL + TILES * D <= 512, "tensor memory");
    static_assert(TOTAL + 1024 <= 227 * 1024, "shared memory of the prompt kernel");
};

// MN-major operand with the 128-byte swizzle: panels of 64 elements (128 bytes) along MN, `panel` bytes apart; groups of
// eight k-rows 1024 bytes apart.
__device__ __forceinline__ uint64_t ap_desc_mn(uint32_t addr, int panel) {
    uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(panel >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void ap_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ uint32_t ap_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// value pair of byte `byte` of word: permute and multiply-add, one each for the integer and the multiply pipe
__device__ __forceinline__ uint32_t ap_lut(uint32_t lut_lane, uint32_t word, int byte) {
    uint32_t v;
    asm("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(__byte_perm(word, 0u, 0x4440 | byte) * 128u + lut_lane));
    return v;
}
__device__ __forceinline__ uint64_t ap_pack2(uint32_t lo, uint32_t hi) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi)); return r; }
__device__ __forceinline__ void ap_unpack2(uint64_t x, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t ap_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t ap_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// One block of rows of one (sequence, kv head), the unit of work.
template <int TILES, int KT> struct ApItem {
    int b, h, r0, rows, row0, n, len, first;
    int tiles;                                                       // 128-row tiles that hold rows
    int lo, hi, start, nk;                                           // keys any row sees: [lo, hi), from place `start` in nk tiles

    // false: no rows
    __device__ __forceinline__ bool get(const Attn4Args &A, int item, int blocks) {
        const int bh = A.sq.batch * A.kv.kv_heads;
        const int blk = item / bh, x = item - blk * bh;
        b = x / A.kv.kv_heads;
        h = x - b * A.kv.kv_heads;
        r0 = (blocks - 1 - blk) * (TILES * 128);                     // rows with many keys first
        A.sq.get(b, row0, n, len);
        rows = n * A.group;
        if (r0 >= rows) return false;
        tiles = TILES == 2 && r0 + 128 < rows ? 2 : 1;
        first = len - n;
        const int i_lo = r0 / A.group, i_hi = min(n - 1, (r0 + TILES * 128 - 1) / A.group);
        hi = max(0, A.causal ? min(len, first + i_hi + 1) : len);
        lo = A.window > 0 ? max(0, first + i_lo + 1 - A.window) : 0;
        start = lo & ~(KV4_GROUP - 1);
        nk = hi > lo ? (hi - start + KT - 1) / KT : 0;
        return true;
    }
};

template <int D, int BS, typename T>
__global__ void __launch_bounds__(AP_THREADS, 1)
attn4_prompt_kernel(const __grid_constant__ Attn4Args A, int items, int blocks) {
    using S = ApSmem<D, BS>;
    constexpr int TILES = S::TILES, KT = S::KT, NB = D / BS, SOFF = KV4_GROUP * (D / 2), HALF = kv4_half_bytes(D, BS);
    constexpr bool BF = !std::is_same<T, __half>::value;
    constexpr uint32_t INF = BF ? 0x7f80u : 0x7c00u;
    using Item = ApItem<TILES, KT>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem), bar = sb + S::BAR;
    const uint32_t k_full = bar + 8, k_empty = bar + 16, v_full = bar + 24, v_empty = bar + 32;
    auto raw_full = [&](int s) { return bar + 40 + 8u * s; };
    auto raw_empty = [&](int s) { return bar + 56 + 8u * s; };
    auto s_full = [&](int t) { return bar + 72 + 8u * t; };
    auto p_full = [&](int t) { return bar + 88 + 8u * t; };
    auto o_done = [&](int t) { return bar + 104 + 8u * t; };
    auto q_full = [&](int t) { return bar + 120 + 8u * t; };
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem + S::BAR + 160);
    volatile uint32_t *abort_flag = tmem_slot + 1, *never = tmem_slot + 2;               // never: stays 0
    volatile float *k_pow = reinterpret_cast<volatile float *>(smem + S::BAR + 176);     // [2]: power of two of a K tile
    volatile int *v_exp = reinterpret_cast<volatile int *>(smem + S::BAR + 192);         // [2]: V's exponent from a tile on

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(k_full, 8); mbar_init(k_empty, 1); mbar_init(v_full, 8); mbar_init(v_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(raw_full(i), 1); mbar_init(raw_empty(i), 8);
            mbar_init(s_full(i), 1); mbar_init(p_full(i), 4); mbar_init(o_done(i), 1); mbar_init(q_full(i), 4);
        }
        *abort_flag = *never = 0;
        fence_mbar_init();
    }
    if (warp == AP_MMA) {
        tmem_alloc(smem_u32((const void *)tmem_slot), 512);
        tmem_relinquish();
    }
    if (warp >= AP_EXPAND && warp < AP_MMA) {
        const float mine = A.code[lane & 15];
        for (int x = warp - AP_EXPAND; x < 256; x += 8) {
            const float c0 = __shfl_sync(0xffffffffu, mine, x & 15), c1 = __shfl_sync(0xffffffffu, mine, x >> 4);
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(sb + (uint32_t)(S::LUT + x * 128 + lane * 4)), "r"(ap_half2(c0, c1)) : "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Every role walks the block's items by itself; what it counts runs on from item to item: key tiles (jj), and tiles
    // of scores per row tile.
#define AP_WAIT(b_, ph_, code_) if (!mbar_wait(b_, ph_, abort_flag)) { atomicExch(&g_attn4_prompt_status, code_); *abort_flag = 1; break; }

    if (warp == AP_LOAD) {
        // ------------------------------------------------------------ codes
        int jj = 0;
        for (int item = blockIdx.x; item < items && !*abort_flag; item += gridDim.x) {
            Item w;
            if (!w.get(A, item, blocks)) continue;
            for (int j = 0; j < w.nk; ++j, ++jj) {
                const int st = jj & 1;
                AP_WAIT(raw_empty(st), ((jj >> 1) & 1) ^ 1, 411);
                const int place = w.start + j * KT + lane * KV4_GROUP;
                const bool want = lane < KT / KV4_GROUP && place < w.hi;
                int page = -1;
                if (want) page = __ldg(A.sq.table + (int64_t)w.b * A.sq.table_ld + (place >> A.kv.page_shift));
                const bool good = want && page >= 0 && page < A.kv.num_pages;
                const uint32_t dst = sb + S::RAW + st * S::CODES + lane * S::GROUP;
                if (want && !good) {
                    // a page outside the cache: its keys are NaN
                    atomicExch(&g_attn4_prompt_status, KV4_BAD_PAGE);
                    for (int i = 0; i < KV4_GROUP * NB; ++i) {
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + SOFF + 2 * i), "h"((uint16_t)0x7fff) : "memory");
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + HALF + SOFF + 2 * i), "h"((uint16_t)0) : "memory");
                    }
                }
                const uint32_t goods = __ballot_sync(0xffffffffu, good);
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(raw_full(st), (uint32_t)(__popc(goods) * S::GROUP));
                __syncwarp();
                if (good) bulk_load_1d(dst, A.kv.group(page, w.h, place), S::GROUP, raw_full(st));
            }
        }
        // no copy may be in flight when the block ends (they are not, unless a wait has run out)
        for (int j = max(0, jj - 2); j < jj; ++j) mbar_wait(raw_full(j & 1), (j >> 1) & 1, never);
    } else if (warp == AP_MMA) {
        // ------------------------------------------------------------ products
        if (lane == 0) {
            const uint32_t idesc_s = umma_idesc_f16(0, 128, KT);
            const uint32_t idesc_o = umma_idesc_f16(0, 128, D) | (1u << 16);             // B is MN-major
            auto scores = [&](int t) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint64_t da = umma_desc_k_sw128(sb + S::Q + (t * S::PANELS + k / 4) * S::Q_PANEL) + 2 * (k & 3);
                    const uint64_t db = umma_desc_k_sw128(sb + S::K + (k / 4) * S::PANEL) + 2 * (k & 3);
                    umma_f16(tmem + S::S_COL + t * 128, da, db, idesc_s, k > 0);
                }
                umma_commit(s_full(t));
            };
            int jj = 0, count[2] = {0, 0}, done[2] = {0, 0};         // key tiles; score tiles and items of either row tile
            for (int item = blockIdx.x; item < items && !*abort_flag; item += gridDim.x) {
                Item w;
                if (!w.get(A, item, blocks)) continue;
                if (w.nk == 0) continue;
                bool ok = false;
                do {
                    AP_WAIT(k_full, jj & 1, 413);
                    AP_WAIT(q_full(0), done[0] & 1, 412);
                    ++done[0];
                    tc_fence_after();
                    scores(0);
                    if (w.tiles == 2) {
                        AP_WAIT(q_full(1), done[1] & 1, 412);
                        ++done[1];
                        tc_fence_after();
                        scores(1);
                    }
                    umma_commit(k_empty);
                    ok = true;
                } while (false);
                for (int j = 0; j < w.nk && ok; ++j, ++jj) {
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        if (t >= w.tiles) break;
                        ok = false;
                        AP_WAIT(p_full(t), count[t] & 1, 414);
                        ++count[t];
                        if (t == 0) { AP_WAIT(v_full, jj & 1, 415); }
                        tc_fence_after();
#pragma unroll
                        for (int k = 0; k < KT / 16; ++k)
                            umma_f16_tmem_a(tmem + S::O_COL + t * D, tmem + S::S_COL + t * 128 + k * 8,
                                            ap_desc_mn(sb + S::V + k * 16 * 128, S::PANEL), idesc_o, j > 0 || k > 0);
                        umma_commit(o_done(t));
                        if (t == w.tiles - 1) umma_commit(v_empty);
                        if (j + 1 < w.nk) {
                            if (t == 0) { AP_WAIT(k_full, (jj + 1) & 1, 416); tc_fence_after(); }
                            scores(t);                               // over P: the MMAs run in the order of their issue
                            if (t == w.tiles - 1) umma_commit(k_empty);
                        }
                        ok = true;
                    }
                }
                if (!ok) break;
            }
        }
    } else if (warp >= AP_EXPAND) {
        // ------------------------------------------------------------ operand tiles from codes
        const int w0 = warp - AP_EXPAND;
        constexpr int CH = D / 32;                                   // 32-channel pieces (16 bytes of codes) of a row
        constexpr int PER = KT * CH / 256;                           // pieces per thread and side
        constexpr int STEP = 256 / CH;                               // tokens from one piece of a thread to its next
        static_assert(STEP % KV4_GROUP == 0, "a thread's pieces have the same place in their groups");
        const uint32_t lut = sb + S::LUT + lane * 4;
        const int tok = (w0 * 32 + lane) / CH, q = lane % CH, panel = q >> 1, half = q & 1;
        // panels are a multiple of 128 bytes apart: lanes of different panels take their 16-byte columns in
        // different orders, so that eight neighbours meet in no bank
        const int turn = D == 128 ? (panel & 1) * 2 : D == 256 ? panel : 0;
        const uint32_t src0 = (tok >> 4) * S::GROUP + (tok & 15) * (D / 2) + q * 16;
        const uint32_t sc0 = (tok >> 4) * S::GROUP + SOFF + 2 * ((tok & 15) * NB + q * 32 / BS);
        uint32_t col[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) col[i] = panel * S::PANEL + tok * 128 + ((((half << 2) | (i ^ turn)) ^ (tok & 7)) << 4);
        int jj = 0;
        for (int item = blockIdx.x; item < items && !*abort_flag; item += gridDim.x) {
            Item w;
            if (!w.get(A, item, blocks)) continue;
            int v_cur = 0;                                           // exponent (biased) that V is brought down by
            for (int j = 0; j < w.nk; ++j, ++jj) {
                const int st = jj & 1, place0 = w.start + j * KT;
                AP_WAIT(raw_full(st), (jj >> 1) & 1, 417);
                const uint32_t raw = sb + S::RAW + st * S::CODES;
                const bool part = place0 < w.lo || place0 + KT > w.hi;
                // largest absmax of the tile's keys and values (bits of a 16-bit type; an infinity or a NaN is the largest)
                uint32_t mk = 0, mv = 0;
                auto scan = [&](uint32_t limit) {
                    mk = mv = 0;
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i) {
                        const int t = lane + 32 * i;
                        if (part && (place0 + t < w.lo || place0 + t >= w.hi)) continue;
                        const uint32_t at = raw + (t >> 4) * S::GROUP + SOFF + (t & 15) * (2 * NB);
#pragma unroll
                        for (int e = 0; e < NB; ++e) {
                            uint16_t x, y;
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at + 2 * e) : "memory");
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(at + HALF + 2 * e) : "memory");
                            const uint32_t xx = x & 0x7fffu, yy = y & 0x7fffu;
                            mk = max(mk, xx < limit ? xx : 0u);
                            mv = max(mv, yy < limit ? yy : 0u);
                        }
                    }
                    mk = __reduce_max_sync(0xffffffffu, mk);
                    mv = __reduce_max_sync(0xffffffffu, mv);
                };
                scan(0x8000u);
                const bool odd = mv >= INF;                          // some value is not finite
                if (mk >= INF || odd) scan(INF);
                auto exponent = [&](uint32_t bits) -> int {
                    const uint16_t x = (uint16_t)bits;
                    const int e = (int)(__float_as_uint(to_f32<T>(*reinterpret_cast<const T *>(&x))) >> 23);
                    return max(9, min(253, e));
                };
                const int ek = exponent(mk), ev = exponent(mv);
                if (j == 0 || ev > v_cur + 6) v_cur = ev;            // V stays under 2^15
                const float down_k = __int_as_float((262 - ek) << 23), down_v = __int_as_float((262 - v_cur) << 23);
                AP_WAIT(k_empty, (jj & 1) ^ 1, 418);
                if (w0 == 0 && lane == 0) { k_pow[st] = __int_as_float((ek - 8) << 23); v_exp[st] = v_cur; }
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    if (side == 1) { AP_WAIT(v_empty, (jj & 1) ^ 1, 419); }
                    const uint32_t tile = sb + (side == 0 ? S::K : S::V);
#pragma unroll
                    for (int it = 0; it < PER; ++it) {
                        const uint32_t src = raw + side * HALF + it * (STEP / KV4_GROUP * S::GROUP);
                        uint32_t c[4];
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
                                     : "r"(src + src0) : "memory");
                        uint16_t sbits;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(sbits) : "r"(src + sc0) : "memory");
                        float s = to_f32<T>(*reinterpret_cast<const T *>(&sbits));
                        if (side == 0) {
                            s *= down_k;
                            if (odd) {                               // it has to reach the rows that see it and no others: through its key
#pragma unroll
                                for (int e = 0; e < NB; ++e) {
                                    uint16_t y;
                                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(src + sc0 - 2 * (q * 32 / BS) + HALF + 2 * e) : "memory");
                                    if ((y & INF) == INF) s = __int_as_float(0x7fc00000);
                                }
                            }
                        } else {
                            s *= down_v;
                            const int place = place0 + tok + it * STEP;
                            if (part && (place < w.lo || place >= w.hi)) s = 0.0f;
                            if (odd && (sbits & INF) == INF) s = 0.0f;
                        }
                        const __half2 s2 = __float2half2_rn(s);
                        if (turn & 1) { uint32_t x = c[0]; c[0] = c[1]; c[1] = x; x = c[2]; c[2] = c[3]; c[3] = x; }
                        if (turn & 2) { uint32_t x = c[0]; c[0] = c[2]; c[2] = x; x = c[1]; c[1] = c[3]; c[3] = x; }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t o[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t p = ap_lut(lut, c[i], e);
                                const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&p), s2);
                                o[e] = *reinterpret_cast<const uint32_t *>(&y);
                            }
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(tile + col[i] + it * (STEP * 128)),
                                         "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(side == 0 ? k_full : v_full);
                        if (side == 1) mbar_arrive(raw_empty(st));
                    }
                }
                if (*abort_flag) break;
            }
        }
    } else if (warp < 4 * TILES) {
        // ------------------------------------------------------------ softmax: one row per thread
        const int t = warp >> 2, rr = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + S::S_COL + t * 128 + lanes, t_o = tmem + S::O_COL + t * D + lanes;
        const uint32_t negate = A.scale_log2 < 0.0f ? 0x80008000u : 0u;   // a negative scale goes into q: maxima stay maxima
        int jj = 0, count = 0;
        bool ok = true;
        for (int item = blockIdx.x; item < items && ok && !*abort_flag; item += gridDim.x) {
            Item w;
            if (!w.get(A, item, blocks)) continue;
            if (t >= w.tiles) { jj += w.nk; continue; }
            const int r = w.r0 + threadIdx.x, i = r / A.group, g = r - i * A.group;
            const bool live = r < w.rows;
            float f = fabsf(A.scale_log2) * attn4_code_unscale(A.quant_type);   // score -> power of two
            if (w.nk > 0) {                                          // (an item without keys has no products: q is not announced)
                const T *src = reinterpret_cast<const T *>(A.q) + (int64_t)(w.row0 + i) * A.q_ts + (int64_t)(w.h * A.group + g) * A.q_hs;
                uint4 x[D / 8];
#pragma unroll
                for (int k = 0; k < D / 8; ++k) {
                    x[k] = make_uint4(0u, 0u, 0u, 0u);
                    if (live) x[k] = __ldg(reinterpret_cast<const uint4 *>(src) + k);
                }
                float down = 1.0f;
                if constexpr (BF) {
                    uint32_t mx = 0;
                    auto upd = [&](uint32_t y) { mx = max(mx, max(y & 0x7fffu, (y >> 16) & 0x7fffu)); };
#pragma unroll
                    for (int k = 0; k < D / 8; ++k) { upd(x[k].x); upd(x[k].y); upd(x[k].z); upd(x[k].w); }
                    const int e = max(1, min(253, (int)(mx >> 7)));
                    down = __int_as_float((254 - e) << 23);
                    f *= __int_as_float(e << 23);
                }
                auto cv = [&](uint32_t y) {
                    y ^= negate;
                    return BF ? ap_half2(__uint_as_float(y << 16) * down, __uint_as_float(y & 0xffff0000u) * down) : y;
                };
#pragma unroll
                for (int k = 0; k < D / 8; ++k) {
                    const uint32_t dst = sb + S::Q + (t * S::PANELS + k / 8) * S::Q_PANEL + rr * 128 + (((k & 7) ^ (rr & 7)) << 4);
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(cv(x[k].x)), "r"(cv(x[k].y)), "r"(cv(x[k].z)), "r"(cv(x[k].w)) : "memory");
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full(t));
            }
            const int lim = live ? (A.causal ? w.first + i + 1 : w.len) : 0, low = A.window > 0 ? lim - A.window : 0;
            // keys that every row of this warp sees: [wh, wl)
            const int wl = __reduce_min_sync(0xffffffffu, live ? lim : 0x7fffffff), wh = __reduce_max_sync(0xffffffffu, live ? low : 0);
            float m = ATTN4_NONE;
            uint64_t l2 = 0;                                         // two partial sums
            int ve = 0;
            for (int j = 0; j < w.nk; ++j, ++jj, ++count) {
                ok = false;
                AP_WAIT(s_full(t), count & 1, 420);
                tc_fence_after();
                const int place0 = w.start + j * KT;
                const float fj = f * k_pow[jj & 1];
                const int vn = v_exp[jj & 1];
                bool bad = false;
                // MASKED: some row of the warp does not see some key of the tile
                auto tile = [&](auto MASKED) {
                    auto hidden = [&](int c) { const int place = place0 + c; return !(place < lim && place >= low); };
                    uint32_t v[32];
                    float mx = __int_as_float(0xff800000);
#pragma unroll
                    for (int c0 = 0; c0 < KT; c0 += 32) {
                        tmem_ld_32x32(t_s + c0, v);
                        tmem_ld_wait();
                        float a0 = mx, a1 = mx;
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            if (MASKED) {
#pragma unroll
                                for (int x = 0; x < 4; ++x) if (hidden(c0 + e + x)) v[e + x] = 0xff800000u;
                            }
                            a0 = fmaxf(a0, fmaxf(__uint_as_float(v[e]), __uint_as_float(v[e + 1])));
                            a1 = fmaxf(a1, fmaxf(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])));
                        }
                        mx = fmaxf(a0, a1);
                    }
                    mx = mx == __int_as_float(0xff800000) ? ATTN4_NONE : mx * fj;
                    float k = 1.0f;
                    if (mx > m + 8.0f) {
                        k = ex2(m - mx);
                        m = mx;
                        float x, y;
                        ap_unpack2(l2, x, y);
                        l2 = ap_pack2(__float_as_uint(x * k), __float_as_uint(y * k));
                    }
                    if (j > 0) {
                        if (vn != ve) k *= __int_as_float(max(0, 127 + ve - vn) << 23);
                        if (__any_sync(0xffffffffu, k != 1.0f)) {
                            if (!mbar_wait(o_done(t), (count - 1) & 1, abort_flag)) { atomicExch(&g_attn4_prompt_status, 421); *abort_flag = 1; bad = true; return; }
                            tc_fence_after();
#pragma unroll 1
                            for (int c0 = 0; c0 < D; c0 += 32) {
                                tmem_ld_32x32(t_o + c0, v);
                                tmem_ld_wait();
#pragma unroll
                                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * k);
                                tmem_st_32x32(t_o + c0, v);
                            }
                            tmem_st_wait();
                        }
                    }
                    ve = vn;
                    const uint64_t f2 = ap_pack2(__float_as_uint(fj), __float_as_uint(fj));
                    const uint64_t b2 = ap_pack2(__float_as_uint(AP_LIFT - m), __float_as_uint(AP_LIFT - m));
#pragma unroll
                    for (int c0 = 0; c0 < KT; c0 += 32) {
                        uint32_t p[16];
                        tmem_ld_32x32(t_s + c0, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float x, y;
                            ap_unpack2(ap_fma2(ap_pack2(v[2 * e], v[2 * e + 1]), f2, b2), x, y);
                            if (MASKED) {
                                if (hidden(c0 + 2 * e)) x = __int_as_float(0xff800000);
                                if (hidden(c0 + 2 * e + 1)) y = __int_as_float(0xff800000);
                            }
                            x = ex2(x);
                            y = ex2(y);
                            l2 = ap_add2(l2, ap_pack2(__float_as_uint(x), __float_as_uint(y)));
                            p[e] = ap_half2(x, y);
                        }
                        ap_tmem_st16(t_s + c0 / 2, p);               // over columns of S that have been read
                    }
                };
                if (place0 < wh || place0 + KT > wl) tile(std::true_type{});
                else tile(std::false_type{});
                if (bad) break;
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(t));
                ok = true;
            }
            if (!ok) break;
            if (w.nk > 0) {
                ok = false;
                AP_WAIT(o_done(t), (count - 1) & 1, 422);
                ok = true;
                tc_fence_after();
            }
            float la, lb;
            ap_unpack2(l2, la, lb);
            const float l = la + lb;
            const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l) * __int_as_float(max(1, ve - 8) << 23) * attn4_code_unscale(A.quant_type);
            const int64_t orow = (int64_t)(w.row0 + i) * A.heads + w.h * A.group + g;
            T *dst = reinterpret_cast<T *>(A.out) + orow * D;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                uint32_t v[32];
                if (w.nk > 0) {
                    tmem_ld_32x32(t_o + c0, v);
                    tmem_ld_wait();
                }
                uint32_t y[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    T pr[2] = {from_f32<T>(0.0f), from_f32<T>(0.0f)};
                    if (l != 0.0f) { pr[0] = from_f32<T>(__uint_as_float(v[2 * e]) * inv); pr[1] = from_f32<T>(__uint_as_float(v[2 * e + 1]) * inv); }
                    y[e] = *reinterpret_cast<const uint32_t *>(pr);
                }
                if (live) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) *reinterpret_cast<uint4 *>(dst + c0 + 8 * e) = make_uint4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
                }
            }
            tc_fence_before();                                       // O has been read before the next item's P is announced
            if (live && A.lse != nullptr) A.lse[orow] = l == 0.0f ? __int_as_float(0xff800000) : (m - AP_LIFT + __log2f(l)) * 0.69314718f;
        }
    }
#undef AP_WAIT
    tc_fence_before();
    __syncthreads();
    if (warp == AP_MMA) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
template <int D, int BS, typename T>
static int ap_launch(const Attn4Args &a, cudaStream_t st) {
    using S = ApSmem<D, BS>;
    constexpr int smem = S::TOTAL + 1024;
    static bool configured[64] = {};
    int dev = 0;
    MPSBNB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        MPSBNB_CUDA_TRY(cudaFuncSetAttribute(attn4_prompt_kernel<D, BS, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const int64_t bh = (int64_t)a.sq.batch * a.kv.kv_heads, blocks = ((int64_t)a.sq.new_tokens * a.group + S::TILES * 128 - 1) / (S::TILES * 128);
    if (bh * blocks > 0x7fffffffll) return MPSBNB_ERR_TOO_LARGE;
    const int items = (int)(bh * blocks), sms = sm_count();
    attn4_prompt_kernel<D, BS, T><<<items < sms ? items : sms, AP_THREADS, smem, st>>>(a, items, (int)blocks);
    return check_launch();
}

int attn4_prompt(const Attn4Args &a, int head_dim, int blocksize, int dtype, cudaStream_t st) {
#define AP_PICK(D, BS) return dtype == MPSBNB_F16 ? ap_launch<D, BS, __half>(a, st) : ap_launch<D, BS, __nv_bfloat16>(a, st)
    if (blocksize == 32) {
        if (head_dim == 64) AP_PICK(64, 32);
        if (head_dim == 128) AP_PICK(128, 32);
        AP_PICK(256, 32);
    }
    if (head_dim == 64) AP_PICK(64, 64);
    if (head_dim == 128) AP_PICK(128, 64);
    AP_PICK(256, 64);
#undef AP_PICK
}

int attn4_prompt_status_fetch(int *out, bool reset) {
    MPSBNB_CUDA_TRY(cudaMemcpyFromSymbol(out, g_attn4_prompt_status, sizeof(int)));
    if (reset) {
        const int zero = 0;
        MPSBNB_CUDA_TRY(cudaMemcpyToSymbol(g_attn4_prompt_status, &zero, sizeof(int)));
    }
    return MPSBNB_OK;
}

}  // namespace mpsbnb
