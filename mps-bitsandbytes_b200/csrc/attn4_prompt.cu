// Attention over the paged 4-bit cache for many query rows per sequence (prompts): out = softmax(scale q K^T) V on the
// 5th-generation tensor cores, K and V expanded from their codes into operand tiles in shared memory.
//
// Floor: the tensor pipe (4 rows keys head_dim operations) and, level with it at head_dim 128, the exponentials (16 a clock
// and SM).  A tile of 256 rows and 128 keys: 2050 clocks for the products, 2050 for the powers, 3200 of shared memory (look-ups of
// codes 1000, expanded operands written 500 and read by the products 1500 - 1700); it takes about 4500.  64 heads on 8 of 128,
// 4096 tokens, causal: 366 us, 0.75 PFLOP/s of what the mask leaves, tensor pipe 39 - 44 % busy; of 64, 303 us, 0.45 (powers and
// expanding cost the same, products half).  When it took 344 us it took 303 without the expanders' arithmetic, 231 without the softmax's,
// 198 without both: what is left is products and hand-overs, and each of the two adds to them through shared memory and issue slots rather
// than by being waited for - P announced by halves, so that its first products begin early, changed nothing.  The roles' code does not
// fit the instruction cache together (1 of 9 stalled warps waits for it): 20 instructions more in a role cost 2 - 3 %.
//
// A block takes 256 rows (or the last 128) of one (sequence, kv head) at a time, long ones first; a row is a (new token,
// head of the group) pair, so all heads of a group share each expanded tile.  Two 128-row tiles A and B alternate: while
// the softmax warps of one work, the tensor core does the other's products.  head_dim 256 takes one tile of 128 rows
// (tensor memory: 256 columns of O), 64 keys at a time and two buffers of S instead.  Roles:
//   warps 0-3, 4-7  softmax of tile A / B, one row per thread: S from tensor memory, P back over S as fp16, the row's sum
//                   in fp32.  The reference m follows the maximum only when that exceeds it by more than 2^8; O stays in
//                   tensor memory and is rescaled only then.
//   warps 8-15      expand a tile of KT keys: byte -> fp16 pair by a table held once per lane, times the block's absmax,
//                   into 128-byte-swizzled panels [KT][64 channels].  For K that is the K-major operand of S = Q K^T,
//                   for V - the same layout read the other way - the MN-major operand of O = P V.  K and V take turns in
//                   a ring of three buffers, so expanding runs ahead of the products.
//   warp 16         issues the MMAs: S_A, S_B, then per key tile O_A += P_A V, S_A(next), O_B += P_B V, S_B(next), on
//                   into the next block of rows without a pause.
//   warp 17         fetches the codes: one bulk copy per group of 16 tokens, two tiles ahead.
//   warps 18, 19    bring the next rows of q as soon as the last products with the present ones have been issued
//                   (head_dim 256: warps 4-7, which have no second tile).
// Where few blocks of rows would leave SMs idle, a block takes an equal run of all their key tiles instead, and partial results are
// joined (attn4.cuh): 8 heads of 1024 rows over 8192 keys 71 us, of 4096 rows over 32768 keys 583.
// Rounding: code * absmax of K and of V and the powers P go to fp16 once each, 2.1e-4 in the root mean square; an fp16 output is then
// off by 4.8e-4 of its size, half a step of its type (its own rounding: 2.1e-4 on average), a bf16 output by 1.76e-3 where its own
// rounding makes 1.66e-3 (24 000 keys).
// Products in TF32 would halve the rate and double the operands.
// fp16 operands hold bf16 caches too: the absmax of a K tile (and, carried along, of the V tiles) is brought near 2^8 by
// a power of two that the scores' factor (and the end of the row, or a rescale of O) takes back.  Blocks of elements that this
// leaves under 2^-14, of which fp16 keeps too few bits, are noticed: their sequence is done again by attn4_decode_kernel, which
// takes any magnitudes side by side, and scores of any size: its launch costs 5 us where it finds nothing to do, the look at the
// magnitudes 0 - 3 %; a prompt of 4096 that is done again takes 4.0 ms.
#include <type_traits>

#include "attn4.cuh"

namespace mpsbnb {

using namespace sm100;

static __device__ int g_attn4_prompt_status = 0;

// P is 2^(x - m + 7): at most 2^15 while the reference m lags by 2^8, and what lies 2^21 below the reference still has
// fp16's full precision.
constexpr float AP_LIFT = 7.0f;
constexpr int AP_EXPAND = 8, AP_EXPANDERS = 8;                       // first expander warp, their number
constexpr int AP_MMA = 16, AP_LOAD = 17, AP_Q = 18, AP_THREADS = 20 * 32;
// Registers: launched with 96 a thread (640 threads); the warpgroups then share them out anew.  (A spilled register costs a
// trip to L2 here: shared memory leaves next to nothing of L1.  head_dim 64 and 128 spill 80 - 116 bytes a thread of the softmax: 1.5 % of
// all instructions.)
constexpr int AP_REGS = 96, AP_REGS_SOFTMAX = 128, AP_REGS_EXPAND = 72, AP_REGS_OTHER = 80;
static_assert(2 * AP_REGS_SOFTMAX + 2 * AP_REGS_EXPAND + AP_REGS_OTHER <= 5 * AP_REGS, "a raise beyond the launch's registers would wait for ever");
template <int N> __device__ __forceinline__ void ap_regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void ap_regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int D, int BS> struct ApSmem {
    static constexpr int TILES = D > 128 ? 1 : 2;                    // 128-row tiles
    static constexpr int KT = D > 128 ? 64 : 128;                    // keys per tile
    static constexpr int PANELS = D / 64, PANEL = KT * 128, Q_PANEL = 128 * 128, BUF = PANELS * PANEL;
    static constexpr int GROUP = 2 * kv4_half_bytes(D, BS), CODES = KT / KV4_GROUP * GROUP;
    static constexpr int NBUF = D > 64 && BS == 32 ? 2 : 3;          // operand buffers (what fits)
    static constexpr int Q_WARPS = TILES == 1 ? 4 : 2;               // that bring q
    static constexpr int Q = 0;
    static constexpr int RING = Q + TILES * PANELS * Q_PANEL;
    static constexpr int LUT = RING + NBUF * BUF;
    static constexpr int RAW = LUT + 256 * 128;
    static constexpr int EXPO = RAW + 2 * CODES;                     // [2][TILES * 128] bytes: power of two that a bf16 row of q was divided by
    static constexpr int BAR = EXPO + 2 * TILES * 128;
    static constexpr int TOTAL = BAR + 368;
    // tensor memory columns
    static constexpr int S_COL = 0, S_STEP = TILES == 2 ? 128 : 64, O_COL = 2 * S_STEP;
    static_assert(O_COL + TILES * D <= 512, "tensor memory");
};

// Matrix descriptors with the 128-byte swizzle, by halves (the upper one is a constant): rows of 128 bytes, groups of
// eight of them 1024 bytes apart.  K-major: a row is one of M or N, 64 elements of K.  MN-major: a row is one of K, 64
// elements of M or N; the next 64 are `panel` bytes on.
constexpr uint32_t AP_DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t ap_desc_k(uint32_t addr) { return (addr & 0x3FFFFu) >> 4 | 1u << 16; }
__device__ __forceinline__ uint32_t ap_desc_mn(uint32_t addr, int panel) { return (addr & 0x3FFFFu) >> 4 | (uint32_t)(panel >> 4) << 16; }
__device__ __forceinline__ void ap_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}\n"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(AP_DESC_HI)
        : "memory");
}
__device__ __forceinline__ void ap_mma_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}\n"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(AP_DESC_HI)
        : "memory");
}
__device__ __forceinline__ void ap_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void ap_tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// 16 lanes (rows) of 32 columns as the products' own registers have them: of each eight columns lane l gets 2 (l % 4) and the
// next, of row l / 4 and then of row l / 4 + 8
__device__ __forceinline__ void ap_tmem_ld_rows(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
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
__device__ __forceinline__ float ap_max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
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
    int slot;                                                        // where the partial result goes; -1: the item is whole

    // key tiles [a, e) of it
    __device__ __forceinline__ void set(const Attn4Args &A, int b_, int h_, int r0_, int a, int e, int slot_) {
        b = b_; h = h_; r0 = r0_; slot = slot_;
        A.sq.get(b, row0, n, len);
        rows = n * A.group;
        tiles = TILES == 2 && r0 + 128 < rows ? 2 : 1;
        first = len - n;
        const int i_lo = r0 / A.group, i_hi = min(n - 1, (r0 + TILES * 128 - 1) / A.group);
        hi = max(0, A.causal ? min(len, first + i_hi + 1) : len);
        lo = A.window > 0 ? max(0, first + i_lo + 1 - A.window) : 0;
        start = lo & ~(KV4_GROUP - 1);
        nk = hi > lo ? (hi - start + KT - 1) / KT : 0;
        nk = max(0, min(nk, e) - a);
        start += a * KT;
        hi = min(hi, start + nk * KT);
    }
};

// The items of a call, blocks of rows from the last of the longest sequence to the first of all: level by level, so that items
// with many keys come first.  Whole warp.
template <int STEP> struct ApList {
    int level, chunk;                                                // block of rows; 32 sequences
    int64_t before;                                                  // items before this chunk of this level
    uint32_t has;                                                    // sequences of the chunk that have a block at this level
    __device__ __forceinline__ void look(const Attn4Args &A) {
        const int b = chunk * 32 + (threadIdx.x & 31);
        int row0, n = 0, len;
        if (b < A.sq.batch) A.sq.get(b, row0, n, len);
        has = __ballot_sync(0xffffffffu, (int64_t)n * A.group > max((int64_t)level * STEP, (int64_t)A.rows_lo));
    }
    __device__ __forceinline__ void begin(const Attn4Args &A, int blocks) { level = blocks - 1; chunk = 0; before = 0; look(A); }
    // item j, at or behind the one found last; false: there are not so many
    __device__ __forceinline__ bool find(const Attn4Args &A, int64_t j, int &b, int &h, int &r0) {
        while (j >= before + __popc(has) * A.kv.kv_heads) {
            before += __popc(has) * A.kv.kv_heads;
            if ((++chunk) * 32 >= A.sq.batch) { chunk = 0; --level; }
            if (level < 0) return false;
            look(A);
        }
        const int off = (int)(j - before), s = off / A.kv.kv_heads;
        h = off - s * A.kv.kv_heads;
        b = chunk * 32 + (int)__fns(has, 0, s + 1);
        r0 = level * STEP;
        return true;
    }
};

// Few items: the key tiles of all, AP_COST more for each item, are cut into equal runs, one per block, in the order of the pairs
// (block of rows, sequence) with a sequence's heads side by side.  Whole warp.
// (An item's rows of q and its end take as long as 4 tiles or so: 10 us.)
constexpr int AP_COST = 4, AP_ALL = 0x7fffffff;
template <int TILES, int KT> struct ApRun {
    int pair, h, nt;                                                 // where we are; the item's key tiles (one dead one if there is no key)
    int a, e;                                                        // tiles of the piece
    int64_t left, per;                                               // units of the run behind the piece; units of every run
    __device__ __forceinline__ static void place(const Attn4Args &A, int blocks, int pair, int &b, int &r0) {
        const int level = pair / A.sq.batch;
        b = pair - level * A.sq.batch;
        r0 = (blocks - 1 - level) * TILES * 128;
    }
    __device__ __forceinline__ static int tiles(const Attn4Args &A, int blocks, int pair) {   // 0: no such item
        if (pair >= blocks * A.sq.batch) return 0;
        int b, r0;
        ApItem<TILES, KT> w;
        place(A, blocks, pair, b, r0);
        w.set(A, b, 0, r0, 0, AP_ALL, 0);
        return r0 < w.rows && w.rows > A.rows_lo ? max(w.nk, 1) : 0;
    }
    __device__ __forceinline__ static int64_t units(const Attn4Args &A, int nt) { return nt > 0 ? (int64_t)(nt + AP_COST) * A.kv.kv_heads : 0; }
    __device__ __forceinline__ bool begin(const Attn4Args &A, int blocks) {
        const int lane = threadIdx.x & 31, pairs = blocks * A.sq.batch;
        int64_t total = 0;
        for (int p = lane; p < pairs; p += 32) total += units(A, tiles(A, blocks, p));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        per = max((total + gridDim.x - 1) / gridDim.x, (int64_t)(AP_COST + 4));
        const int64_t t0 = min(total, blockIdx.x * per), t1 = min(total, t0 + per);
        left = t1 - t0;
        if (left == 0) return false;
        int64_t base = 0, inc;
        int mine;
        for (int p0 = 0;; p0 += 32) {
            if (p0 >= pairs) return false;                           // (lengths that change under a running kernel)
            mine = tiles(A, blocks, p0 + lane);
            inc = units(A, mine);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += up;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, base + inc > t0);
            if (hit != 0) {
                const int l = __ffs(hit) - 1;
                pair = p0 + l;
                nt = __shfl_sync(0xffffffffu, mine, l);
                base += __shfl_sync(0xffffffffu, inc, l) - units(A, nt);
                break;
            }
            base += __shfl_sync(0xffffffffu, inc, 31);
        }
        h = (int)((t0 - base) / (nt + AP_COST));
        take((int)(t0 - base - (int64_t)h * (nt + AP_COST)));
        return e > 0 || next(A, blocks);
    }
    __device__ __forceinline__ void take(int from) {                 // the piece that begins `from` units into its item
        const int to = (int)min((int64_t)(nt + AP_COST), from + left);
        left -= to - from;
        a = max(0, from - AP_COST);
        e = max(0, to - AP_COST);
    }
    __device__ __forceinline__ bool next(const Attn4Args &A, int blocks) {
        do {
            if (left == 0) return false;
            if (++h == A.kv.kv_heads) {
                h = 0;
                do {
                    if (++pair >= blocks * A.sq.batch) return false;
                    nt = tiles(A, blocks, pair);
                } while (nt == 0);
            }
            take(0);
        } while (e == 0);
        return true;
    }
};

template <int D, int BS, typename T>
__global__ void __launch_bounds__(AP_THREADS, 1)
attn4_prompt_kernel(const __grid_constant__ Attn4Args A, int split) {
    using S = ApSmem<D, BS>;
    constexpr int TILES = S::TILES, KT = S::KT, NB = D / BS, SOFF = KV4_GROUP * (D / 2), HALF = kv4_half_bytes(D, BS);
    constexpr bool BF = !std::is_same<T, __half>::value;
    constexpr uint32_t INF = BF ? 0x7f80u : 0x7c00u, FLOOR = BF ? 0x322cu : 0u;   // of 16-bit absmax; FLOOR: the quantiser's 1e-8
    using Item = ApItem<TILES, KT>;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t sb = smem_u32(smem), bar = sb + S::BAR;
    if ((sb & 1023u) != 0) {                                         // the swizzle counts on it
        if (threadIdx.x == 0) {                                      // (nothing to join, everything to be done again)
            atomicExch(&g_attn4_prompt_status, 410);
            if (split) attn4_join<D, TILES * 128>(A.ws, gridDim.x)[blockIdx.x].n = 0;
            A.wide[blockIdx.x] = 0xffffffffu;
        }
        return;
    }
    auto buf_full = [&](int s) { return bar + 8u * s; };             // [3]
    auto buf_empty = [&](int s) { return bar + 24 + 8u * s; };       // [3]
    auto raw_full = [&](int s) { return bar + 48 + 8u * s; };        // [2] each from here on
    auto raw_empty = [&](int s) { return bar + 64 + 8u * s; };
    auto s_full = [&](int s) { return bar + 80 + 8u * s; };          // by buffer of S: the row tile, or (one row tile) turn about
    auto p_full = [&](int s) { return bar + 96 + 8u * s; };
    auto o_done = [&](int s) { return bar + 112 + 8u * s; };         // by buffer of S
    auto q_full = [&](int t) { return bar + 128 + 8u * t; };
    auto q_empty = [&](int t) { return bar + 144 + 8u * t; };
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem + S::BAR + 160);
    volatile uint32_t *abort_flag = tmem_slot + 1, *never = tmem_slot + 2;               // never: stays 0
    uint32_t *wide = reinterpret_cast<uint32_t *>(smem + S::BAR + 172);
    volatile float *k_pow = reinterpret_cast<volatile float *>(smem + S::BAR + 176);     // [4]: power of two of a K tile
    volatile int *v_exp = reinterpret_cast<volatile int *>(smem + S::BAR + 192);         // [4]: V's exponent from a tile on
    volatile uint8_t *q_exp = smem + S::EXPO;
    volatile int *queue = reinterpret_cast<volatile int *>(smem + S::BAR + 208);         // [4][6]: items (sequence, or -1; head; row; key tiles; slot)
    auto item_full = [&](int s) { return bar + 304 + 8u * s; };      // [4] each
    auto item_empty = [&](int s) { return bar + 336 + 8u * s; };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::NBUF; ++i) { mbar_init(buf_full(i), AP_EXPANDERS); mbar_init(buf_empty(i), 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(raw_full(i), 1); mbar_init(raw_empty(i), AP_EXPANDERS);
            mbar_init(s_full(i), 1); mbar_init(p_full(i), 4); mbar_init(o_done(i), 1);
            mbar_init(q_full(i), S::Q_WARPS); mbar_init(q_empty(i), 1);
        }
        for (int i = 0; i < 4; ++i) { mbar_init(item_full(i), 1); mbar_init(item_empty(i), 4 * TILES + AP_EXPANDERS + 1 + S::Q_WARPS); }   // (1: the issuer)
        *abort_flag = *never = *wide = 0;
        fence_mbar_init();
    }
    if (warp == AP_MMA) {
        tmem_alloc(smem_u32((const void *)tmem_slot), 512);
        tmem_relinquish();
    }
    if (warp >= AP_EXPAND && warp < AP_MMA) {
        const float mine = A.code[lane & 15];
        for (int x = warp - AP_EXPAND; x < 256; x += AP_EXPANDERS) {
            const float c0 = __shfl_sync(0xffffffffu, mine, x & 15), c1 = __shfl_sync(0xffffffffu, mine, x >> 4);
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(sb + (uint32_t)(S::LUT + x * 128 + lane * 4)), "r"(ap_half2(c0, c1)) : "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // The loader finds the block's items - every second time round in the opposite direction, which evens the blocks out - and
    // queues them for the other roles.  What a role counts (key tiles, operands, tiles of scores) runs on from item to item.
    int turn_ = 0;                                                   // of the queue
    // the next item; false: no more.  Whole warp (or the one thread of the issuer)
    auto next_item = [&](Item &w, bool one) -> bool {
        const int s = turn_ & 3;
        if (!mbar_wait(item_full(s), (turn_ >> 2) & 1, abort_flag)) { atomicExch(&g_attn4_prompt_status, 424); *abort_flag = 1; return false; }
        volatile int *it = queue + 6 * s;
        const int b = it[0], h = it[1], r0 = it[2], a = it[3], e = it[4], slot = it[5];
        if (!one) __syncwarp();
        if (one || lane == 0) mbar_arrive(item_empty(s));
        ++turn_;
        if (b < 0) return false;
        w.set(A, b, h, r0, a, e, slot);
        return true;
    };
#define AP_WAIT(b_, ph_, code_) if (!mbar_wait(b_, ph_, abort_flag)) { atomicExch(&g_attn4_prompt_status, code_); *abort_flag = 1; break; }

    // ------------------------------------------------------------ q: 16 bytes per lane, LPR lanes a row
    // Straight into the swizzled panels by asynchronous copies, all of a lane's under way at once; a bf16 row is then turned into fp16 where it lies.  Lane l finds where the
    // warp's rows l, l + 32 lie and hands that to the lanes that copy them.
    auto bring_q = [&](int part) {
        constexpr int LPR = D / 8, ROWS = 32 / LPR, STEPS = 32 / ROWS;   // rows a step, steps for 32 rows
        constexpr int MINE = 128 / S::Q_WARPS, PARTS = MINE / 32;    // rows of this warp, lanes' rows
        const uint32_t negate = A.scale_log2 < 0.0f ? 0x80008000u : 0u;   // a negative scale goes into q: maxima stay maxima
        const int k = lane % LPR, my = lane / LPR, base = part * MINE;
        int count[2] = {0, 0};
        Item w;
        while (!*abort_flag && next_item(w, false)) {
            if (w.nk == 0) continue;
            uint64_t src[TILES][PARTS];                              // 0: no such row
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int x = 0; x < PARTS; ++x) {
                    const int r = w.r0 + t * 128 + base + x * 32 + lane, i = r / A.group, g = r - i * A.group;
                    src[t][x] = r < w.rows ? reinterpret_cast<uint64_t>(reinterpret_cast<const T *>(A.q) + (int64_t)(w.row0 + i) * A.q_ts + (int64_t)(w.h * A.group + g) * A.q_hs) : 0;
                }
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                if (t >= w.tiles) break;
                auto dest = [&](int rr) { return sb + S::Q + (t * S::PANELS + k / 8) * S::Q_PANEL + rr * 128 + (((k & 7) ^ (rr & 7)) << 4); };
                AP_WAIT(q_empty(t), (count[t] & 1) ^ 1, 423);
#pragma unroll
                for (int x = 0; x < PARTS; ++x)
#pragma unroll 16
                    for (int s = 0; s < STEPS; ++s) {
                        const uint64_t from = __shfl_sync(0xffffffffu, src[t][x], s * ROWS + my);
                        // (no bytes read, 16 zeros written where there is no row)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dest(base + x * 32 + s * ROWS + my)),
                                     "l"(from != 0 ? from + k * 16 : reinterpret_cast<uint64_t>(A.q)), "r"(from != 0 ? 16 : 0) : "memory");
                    }
                asm volatile("cp.async.wait_all;" ::: "memory");
                if (BF || negate != 0) {
                    // a row to a lane from here on: eight lanes' columns lie in eight different banks' places by the swizzle, and
                    // nothing waits for a shuffle behind the expanders' look-ups
                    __syncwarp();
#pragma unroll 1
                    for (int x = 0; x < PARTS; ++x) {
                        const int rr = base + x * 32 + lane;
                        const uint32_t row = sb + S::Q + t * S::PANELS * S::Q_PANEL + rr * 128;
                        auto at = [&](int c) { return row + (c >> 3) * S::Q_PANEL + (((c & 7) ^ (rr & 7)) << 4); };
                        auto load = [&](int c) {
                            uint4 v;
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at(c)));
                            return v;
                        };
                        uint32_t e2 = 0;
                        if constexpr (BF) {
                            uint32_t m2 = 0;                         // largest magnitudes of the even and odd channels
#pragma unroll 8
                            for (int c = 0; c < LPR; ++c) {
                                const uint4 v = load(c);
                                m2 = __vmaxu2(m2, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
                            }
                            // Less an exponent that brings the row's largest to 2^15 (an infinity or a NaN stays one), two channels
                            // at a time: fp16's bits are then bf16's, three places up.  Parts below 2^-29 of the largest go to
                            // zero, or lose bits.
                            const uint32_t e = max(30u, min(254u, max(m2 & 0xffffu, m2 >> 16) >> 7)) - 30;
                            q_exp[(count[t] & 1) * (TILES * 128) + t * 128 + rr] = (uint8_t)(e + 15);   // of 2^(e - 112), as in fp32
                            e2 = e * 0x00800080u;
                        }
#pragma unroll 4
                        for (int c = 0; c < LPR; ++c) {
                            const uint4 v = load(c);
                            auto cv = [&](uint32_t y) {
                                if constexpr (BF) return ((__vmaxu2(y & 0x7fff7fffu, e2) - e2) << 3) | ((y ^ negate) & 0x80008000u);
                                else return y ^ negate;
                            };
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at(c)), "r"(cv(v.x)), "r"(cv(v.y)), "r"(cv(v.z)), "r"(cv(v.w)));
                        }
                    }
                }
                ++count[t];
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full(t));
            }
        }
    };

    if (warp >= AP_MMA) {
        ap_regs_down<AP_REGS_OTHER>();
        if (warp == AP_LOAD) {
            // -------------------------------------------------------- codes
            int jj = 0;
            ApList<TILES * 128> list;
            ApRun<TILES, KT> run;
            Attn4Join *join = attn4_join<D, TILES * 128>(A.ws, gridDim.x) + blockIdx.x;
            bool more = true;
            const int blocks = (A.sq.longest() * A.group + TILES * 128 - 1) / (TILES * 128);   // of the longest sequence
            if (split) {
                if (lane == 0) join->n = 0;
                __syncwarp();
                more = run.begin(A, blocks);
            } else {
                list.begin(A, blocks);
            }
            for (int turn = 0; !*abort_flag; ++turn) {
                int b = -1, h = 0, r0 = 0, first = 0, end = AP_ALL, slot = -1;
                if (split) {
                    if (more) {
                        run.place(A, blocks, run.pair, b, r0);
                        h = run.h; first = run.a; end = run.e;
                        if (first > 0 || end < run.nt) {
                            slot = turn == 0 ? 0 : 1;                // (a piece between the first and the last is whole)
                            if (first == 0 && lane == 0) {
                                int row0, n, len;
                                A.sq.get(b, row0, n, len);
                                join->slot = slot;
                                join->row0 = row0; join->rows = n * A.group; join->r = r0 / (TILES * 128); join->h = h;
                                join->n = 1 + (int)((run.nt - end + run.per - 1) / run.per);
                            }
                        }
                        more = run.next(A, blocks);
                    }
                } else if (!list.find(A, (int64_t)turn * gridDim.x + (turn & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x), b, h, r0)) {
                    b = -1;
                }
                const int qs = turn & 3;
                AP_WAIT(item_empty(qs), ((turn >> 2) & 1) ^ 1, 425);
                if (lane == 0) {
                    volatile int *it = queue + 6 * qs;
                    it[0] = b; it[1] = h; it[2] = r0; it[3] = first; it[4] = end; it[5] = slot;
                    mbar_arrive(item_full(qs));
                }
                if (b < 0) break;
                Item w;
                w.set(A, b, h, r0, first, end, slot);
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
        } else if (warp >= AP_Q) {
            if constexpr (TILES == 2) bring_q(warp - AP_Q);
        } else if (elect_one()) {
            // -------------------------------------------------------- products
            const uint32_t idesc_s = umma_idesc_f16(0, 128, KT);
            const uint32_t idesc_o = umma_idesc_f16(0, 128, D) | (1u << 16);             // B is MN-major
            int slot = 0; uint32_t ring_phase = 0;                   // operand buffer that comes next, in the order K, V, K, V, ...
            int nq[2] = {0, 0}, np[2] = {0, 0}, ns = 0;              // items begun, score tiles done (by row tile); score tiles begun
            auto step = [&]() { if (++slot == S::NBUF) { slot = 0; ring_phase ^= 1; } };
            auto scores = [&](int t, int buf, bool last) {           // S = Q_t K^T into its buffer
                const int s = TILES == 2 ? t : ns & 1;
                const uint32_t da = ap_desc_k(sb + S::Q + t * S::PANELS * S::Q_PANEL), db = ap_desc_k(sb + S::RING + buf * S::BUF);
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    ap_mma(tmem + S::S_COL + s * S::S_STEP, da + (k / 4) * (S::Q_PANEL >> 4) + 2 * (k & 3), db + (k / 4) * (S::PANEL >> 4) + 2 * (k & 3), idesc_s, k > 0);
                umma_commit(s_full(s));
                if (last) umma_commit(q_empty(t));                   // the item's last products with q
                ++ns;
            };
            auto values = [&](int t, int s, int buf, bool first) {   // O_t (+)= P V
                const uint32_t db = ap_desc_mn(sb + S::RING + buf * S::BUF, S::PANEL);
#pragma unroll
                for (int k = 0; k < KT / 16; ++k)
                    ap_mma_tmem(tmem + S::O_COL + t * D, tmem + S::S_COL + s * S::S_STEP + k * 8, db + k * (16 * 128 >> 4), idesc_o, !first || k > 0);
                umma_commit(o_done(s));
            };
            Item cur, nxt;
            auto fetch = [&](Item &w) -> bool {                      // next item with keys
                while (next_item(w, true))
                    if (w.nk > 0) return true;
                return false;
            };
            bool more = fetch(nxt), ok = true, begun = false;
            // the first scores of `nxt` for row tile t
            auto begin = [&](int t) -> bool {
                do {
                    AP_WAIT(q_full(t), nq[t] & 1, 412);
                    if (t == 0) { AP_WAIT(buf_full(slot), ring_phase, 413); }
                    ++nq[t];
                    tc_fence_after();
                    scores(t, slot, nxt.nk == 1);
                    if (t == nxt.tiles - 1) { umma_commit(buf_empty(slot)); step(); }
                    return true;
                } while (false);
                return false;
            };
            while (more && ok) {
                if (!begun) {
                    for (int t = 0; t < nxt.tiles && ok; ++t) ok = begin(t);
                    if (!ok) break;
                }
                cur = nxt;
                more = false;
                begun = false;
                for (int j = 0; j < cur.nk && ok; ++j) {
                    const bool last = j == cur.nk - 1;
                    if (last) more = fetch(nxt);
                    if (TILES == 2) {
                        const int vbuf = slot; const uint32_t vphase = ring_phase;   // V(j); the K after it is next
                        step();
                        const int kbuf = slot; const uint32_t kphase = ring_phase;
                        for (int t = 0; t < 2 && ok; ++t) {
                            if (t < cur.tiles) {
                                ok = false;
                                AP_WAIT(p_full(t), np[t] & 1, 414);
                                if (t == 0) { AP_WAIT(buf_full(vbuf), vphase, 415); }
                                ++np[t];
                                tc_fence_after();
                                values(t, t, vbuf, j == 0);
                                if (t == cur.tiles - 1) umma_commit(buf_empty(vbuf));
                                ok = true;
                                if (!last) {
                                    ok = false;
                                    if (t == 0) { AP_WAIT(buf_full(kbuf), kphase, 416); tc_fence_after(); }
                                    scores(t, kbuf, j + 2 == cur.nk);   // over P: the MMAs run in the order of their issue
                                    if (t == cur.tiles - 1) { umma_commit(buf_empty(kbuf)); step(); }
                                    ok = true;
                                }
                            }
                            if (last && more && t < nxt.tiles) { ok = begin(t); begun = true; }
                        }
                    } else {
                        // S has two buffers: the next scores go before this tile's products with V
                        const int s = (ns - 1) & 1, vbuf = slot; const uint32_t vphase = ring_phase;
                        step();
                        ok = false;
                        if (!last) {
                            AP_WAIT(buf_full(slot), ring_phase, 416);
                            tc_fence_after();
                            scores(0, slot, j + 2 == cur.nk);
                            umma_commit(buf_empty(slot));
                            step();
                        }
                        AP_WAIT(p_full(s), (np[0] >> 1) & 1, 414);
                        AP_WAIT(buf_full(vbuf), vphase, 415);
                        ++np[0];
                        tc_fence_after();
                        values(0, s, vbuf, j == 0);
                        umma_commit(buf_empty(vbuf));
                        ok = true;
                        if (last && more) { ok = begin(0); begun = true; }
                    }
                }
            }
        }
    } else if (warp >= AP_EXPAND) {
        ap_regs_down<AP_REGS_EXPAND>();
        // ------------------------------------------------------------ operand tiles from codes
        const int w0 = warp - AP_EXPAND;
        constexpr int CH = D / 32;                                   // 32-channel pieces (16 bytes of codes) of a row
        constexpr int PER = KT * CH / (AP_EXPANDERS * 32);           // pieces per thread and side
        constexpr int STEP = AP_EXPANDERS * 32 / CH;                               // tokens from one piece of a thread to its next
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
        int jj = 0, slot = 0; uint32_t ring_phase = 0;
        Item w;
        while (!*abort_flag && next_item(w, false)) {
            int v_cur = 0;                                           // exponent (biased) that V is brought down by
            for (int j = 0; j < w.nk; ++j, ++jj) {
                const int st = jj & 1, place0 = w.start + j * KT;
                AP_WAIT(raw_full(st), (jj >> 1) & 1, 417);
                const uint32_t raw = sb + S::RAW + st * S::CODES;
                const bool part = place0 < w.lo || place0 + KT > w.hi;
                // largest absmax of the tile's keys and values (bits of a 16-bit type; an infinity or a NaN is the largest)
                uint32_t mk = 0, mv = 0;
                {
                    uint32_t k2 = 0, v2 = 0;                         // two at a time
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i) {
                        const int t = lane + 32 * i;
                        if (part && (place0 + t < w.lo || place0 + t >= w.hi)) continue;
                        const uint32_t at = raw + (t >> 4) * S::GROUP + SOFF + (t & 15) * (2 * NB);
#pragma unroll
                        for (int e = 0; e < (NB + 1) / 2; ++e) {
                            uint32_t x, y;
                            if constexpr (NB == 1) {
                                uint16_t x1, y1;
                                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x1) : "r"(at));
                                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y1) : "r"(at + HALF));
                                x = x1; y = y1;
                            } else {
                                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at + 4 * e));
                                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(y) : "r"(at + HALF + 4 * e));
                            }
                            k2 = __vmaxu2(k2, x & 0x7fff7fffu);
                            v2 = __vmaxu2(v2, y & 0x7fff7fffu);
                        }
                    }
                    mk = __reduce_max_sync(0xffffffffu, max(k2 & 0xffffu, k2 >> 16));
                    mv = __reduce_max_sync(0xffffffffu, max(v2 & 0xffffu, v2 >> 16));
                }
                const bool odd = mv >= INF;                          // some value is not finite
                if (mk >= INF || odd) {                              // the largest of those that are
                    mk = mv = 0;
#pragma unroll 1
                    for (int t = lane; t < KT; t += 32) {
                        if (part && (place0 + t < w.lo || place0 + t >= w.hi)) continue;
                        const uint32_t at = raw + (t >> 4) * S::GROUP + SOFF + (t & 15) * (2 * NB);
#pragma unroll 1
                        for (int e = 0; e < NB; ++e) {
                            uint16_t x, y;
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at + 2 * e));
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(at + HALF + 2 * e));
                            const uint32_t xx = x & 0x7fffu, yy = y & 0x7fffu;
                            mk = max(mk, xx < INF ? xx : 0u);
                            mv = max(mv, yy < INF ? yy : 0u);
                        }
                    }
                    mk = __reduce_max_sync(0xffffffffu, mk);
                    mv = __reduce_max_sync(0xffffffffu, mv);
                }
                auto exponent = [&](uint32_t bits) -> int {
                    const uint16_t x = (uint16_t)bits;
                    const int e = (int)(__float_as_uint(to_f32<T>(*reinterpret_cast<const T *>(&x))) >> 23);
                    return max(9, min(253, e));
                };
                const int ek = exponent(mk), ev = exponent(mv);
                if (j == 0 || ev > v_cur + 6) v_cur = ev;            // V stays under 2^15
                const float down_k = __int_as_float((262 - ek) << 23), down_v = __int_as_float((262 - v_cur) << 23);
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    uint32_t c[PER][4];
                    uint16_t sbits[PER];
#pragma unroll
                    for (int it = 0; it < PER; ++it) {
                        const uint32_t src = raw + side * HALF + it * (STEP / KV4_GROUP * S::GROUP);
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(c[it][0]), "=r"(c[it][1]), "=r"(c[it][2]), "=r"(c[it][3]) : "r"(src + src0));
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(sbits[it]) : "r"(src + sc0));
                    }
                    AP_WAIT(buf_empty(slot), ring_phase ^ 1, 418);
                    float sc[PER], low = __int_as_float(0x7f800000);
#pragma unroll
                    for (int it = 0; it < PER; ++it) {
                        sc[it] = to_f32<T>(*reinterpret_cast<const T *>(&sbits[it])) * (side == 0 ? down_k : down_v);
                        low = fminf(low, sc[it]);
                    }
                    if (low < 0x1p-14f) {
#pragma unroll
                        for (int it = 0; it < PER; ++it) {
                            const int place = place0 + tok + it * STEP;
                            if (sc[it] < 0x1p-14f && sbits[it] > FLOOR && place >= w.lo && place < w.hi) atomicOr(wide, 1u << (w.b & 31));
                        }
                    }
                    if (side == 0 && w0 == 0 && lane == 0) { k_pow[jj & 3] = __int_as_float((ek - 8) << 23); v_exp[jj & 3] = v_cur; }
                    const uint32_t tile = sb + S::RING + slot * S::BUF;
#pragma unroll
                    for (int it = 0; it < PER; ++it) {
                        float s = sc[it];
                        if (side == 0) {
                            if (odd) {                               // it has to reach the rows that see it and no others: through its key
#pragma unroll
                                for (int e = 0; e < NB; ++e) {
                                    uint16_t y;
                                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(raw + it * (STEP / KV4_GROUP * S::GROUP) + sc0 - 2 * (q * 32 / BS) + HALF + 2 * e));
                                    if ((y & INF) == INF) s = __int_as_float(0x7fc00000);
                                }
                            }
                        } else {
                            const int place = place0 + tok + it * STEP;
                            if (part && (place < w.lo || place >= w.hi)) s = 0.0f;
                            if (odd && (sbits[it] & INF) == INF) s = 0.0f;
                        }
                        const __half2 s2 = __float2half2_rn(s);
                        if (side == 0) {
                            if (turn & 1) { uint32_t x = c[it][0]; c[it][0] = c[it][1]; c[it][1] = x; x = c[it][2]; c[it][2] = c[it][3]; c[it][3] = x; }
                            if (turn & 2) { uint32_t x = c[it][0]; c[it][0] = c[it][2]; c[it][2] = x; x = c[it][1]; c[it][1] = c[it][3]; c[it][3] = x; }
                        }
                        // K: 16 bytes are the eight channels of a word.  V: one byte of each of the four words, so that column
                        // 8 e + 2 i + (0, 1) of O is channel 8 i + 2 e + (0, 1) of 32.
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t o[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t p = side == 0 ? ap_lut(lut, c[it][i], e) : ap_lut(lut, c[it][e], i ^ turn);
                                const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&p), s2);
                                o[e] = *reinterpret_cast<const uint32_t *>(&y);
                            }
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(tile + col[i] + it * (STEP * 128)),
                                         "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]));
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(buf_full(slot));
                        if (side == 1) mbar_arrive(raw_empty(st));
                    }
                    if (++slot == S::NBUF) { slot = 0; ring_phase ^= 1; }
                }
                if (*abort_flag) break;
            }
        }
    } else if (TILES == 1 && warp >= 4) {
        ap_regs_down<AP_REGS_OTHER>();
        if constexpr (TILES == 1) bring_q(warp - 4);                 // (there is no second row tile)
    } else {
        ap_regs_up<AP_REGS_SOFTMAX>();
        // ------------------------------------------------------------ softmax: one row per thread
        const int t = warp >> 2, rr = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_o = tmem + S::O_COL + t * D + lanes;
        int jj = 0, count = 0, nq = 0;                               // key tiles; score tiles and items of this row tile
        bool ok = true;
        Item w;
        while (ok && !*abort_flag && next_item(w, false)) {
            if (t >= w.tiles) { jj += w.nk; continue; }
            const int r = w.r0 + t * 128 + rr, i = r / A.group, g = r - i * A.group;
            const bool live = r < w.rows;
            const int lim = live ? (A.causal ? w.first + i + 1 : w.len) : 0, low = A.window > 0 ? lim - A.window : 0;
            // keys that every row of this warp sees: [wh, wl)
            const int wl = __reduce_min_sync(0xffffffffu, live ? lim : 0x7fffffff), wh = __reduce_max_sync(0xffffffffu, live ? low : 0);
            float m = ATTN4_NONE, f = fabsf(A.scale_log2) * attn4_code_unscale(A.quant_type);   // f: score -> power of two
            uint64_t l2 = 0;                                         // two partial sums
            int ve = 0;
            for (int j = 0; j < w.nk; ++j, ++jj, ++count) {
                ok = false;
                const int s = TILES == 2 ? t : count & 1;
                const uint32_t t_s = tmem + S::S_COL + s * S::S_STEP + lanes;
                AP_WAIT(s_full(s), (TILES == 2 ? count : count >> 1) & 1, 420);
                tc_fence_after();
                if (BF && j == 0) f *= __int_as_float((int)q_exp[(nq & 1) * (TILES * 128) + t * 128 + rr] << 23);   // (q was there before its products)
                const int place0 = w.start + j * KT;
                const float fj = fmaxf(f * k_pow[jj & 3], 0x1p-126f);        // scale 0: -inf * fj has to stay -inf
                const int vn = v_exp[jj & 3];
                const bool part = place0 < wh || place0 + KT > wl;   // some row of the warp does not see some key of the tile
                const int seen_lo = low - place0, seen_hi = lim - place0;
                auto load = [&](uint32_t (&v)[32], int c0) { tmem_ld_32x32(t_s + c0, v); };
                auto mask = [&](uint32_t (&v)[32], int c0) {
                    if (part) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) if (c0 + e < seen_lo || c0 + e >= seen_hi) v[e] = 0xff800000u;
                    }
                };
                float a0 = __int_as_float(0xff800000), a1 = a0;
                auto maximum = [&](const uint32_t (&v)[32]) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        a0 = ap_max3(a0, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
                        a1 = ap_max3(a1, __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
                    }
                };
                // the first 64 columns are read twice (for the maximum, for P), the others kept
                uint32_t u[2][32], v[2][32];
                if constexpr (KT == 128) {
                    load(u[0], 0); load(u[1], 32);
                    tmem_ld_wait();
                    mask(u[0], 0); mask(u[1], 32);
                    maximum(u[0]); maximum(u[1]);
                }
                load(v[0], KT - 64); load(v[1], KT - 32);
                tmem_ld_wait();
                mask(v[0], KT - 64); mask(v[1], KT - 32);
                maximum(v[0]); maximum(v[1]);
                a0 = fmaxf(a0, a1);
                const float top = a0 == __int_as_float(0xff800000) ? ATTN4_NONE : a0 * fj;
                float k = 1.0f;
                if (top > m + 8.0f) {
                    k = ex2(m - top);
                    m = top;
                    if (fabsf(top) >= ATTN4_FAR) atomicOr(wide, 1u << (w.b & 31));
                }
                const uint64_t f2 = ap_pack2(__float_as_uint(fj), __float_as_uint(fj));
                const uint64_t b2 = ap_pack2(__float_as_uint(AP_LIFT - m), __float_as_uint(AP_LIFT - m));
                uint64_t add = 0;
                auto powers = [&](const uint32_t (&x)[32], uint32_t (&p)[16]) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float y, z;
                        ap_unpack2(ap_fma2(ap_pack2(x[2 * e], x[2 * e + 1]), f2, b2), y, z);
                        y = ex2(y);
                        z = ex2(z);
                        add = ap_add2(add, ap_pack2(__float_as_uint(y), __float_as_uint(z)));
                        p[e] = ap_half2(y, z);
                    }
                };
                uint32_t p0[16], p1[16];
                powers(v[0], p0); powers(v[1], p1);
                if constexpr (KT == 128) {
#pragma unroll
                    for (int c0 = 0; c0 < 64; c0 += 32) {
                        uint32_t p2[16];
                        load(u[0], c0);
                        tmem_ld_wait();
                        mask(u[0], c0);
                        powers(u[0], p2);
                        ap_tmem_st16(t_s + c0 / 2, p2);              // P, over S
                    }
                }
                ap_tmem_st16(t_s + (KT - 64) / 2, p0);
                ap_tmem_st16(t_s + (KT - 32) / 2, p1);
                {
                    float x, y, ax, ay;
                    ap_unpack2(l2, x, y);
                    ap_unpack2(add, ax, ay);
                    l2 = ap_pack2(__float_as_uint(fmaf(x, k, ax)), __float_as_uint(fmaf(y, k, ay)));
                }
                if (j > 0) {
                    if (vn != ve) k *= __int_as_float(max(0, 127 + ve - vn) << 23);
                    if (__any_sync(0xffffffffu, k != 1.0f)) {
                        AP_WAIT(o_done(TILES == 2 ? t : s ^ 1), (TILES == 2 ? count - 1 : (count - 1) >> 1) & 1, 421);
                        tc_fence_after();
#pragma unroll 1
                        for (int c0 = 0; c0 < D; c0 += 16) {
                            uint32_t x[16];
                            ap_tmem_ld16(t_o + c0, x);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * k);
                            ap_tmem_st16(t_o + c0, x);
                        }
                    }
                }
                ve = vn;
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(s));
                ok = true;
            }
            if (!ok) break;
            if (w.nk > 0) {
                ++nq;
                ok = false;
                // (with one row tile the products may be two tiles behind the scores: hence a barrier for each buffer)
                AP_WAIT(o_done(TILES == 2 ? t : (count - 1) & 1), (TILES == 2 ? count - 1 : (count - 1) >> 1) & 1, 422);
                ok = true;
                tc_fence_after();
            }
            float la, lb;
            ap_unpack2(l2, la, lb);
            const float l = la + lb;
            // a partial result: sums as they are, and the reference
            const float up = w.nk > 0 ? __int_as_float(max(1, ve - 8) << 23) * attn4_code_unscale(A.quant_type) : 0.0f;
            const float inv = l == 0.0f ? 0.0f : w.slot < 0 ? __fdividef(1.0f, l) * up : up * ATTN4_SUM;
            // Four lanes take 32 channels (64 bytes) of a row, eight rows at a time: with 16 bytes of 32 rows each, stores kept the
            // load and store unit busy 4 times as long.  (The order that V's channels have in O makes a lane's eight neighbours.)
            float *const part = attn4_partial<D, TILES * 128>(A.ws, blockIdx.x, max(w.slot, 0));
            const int64_t orow = !live ? -1 : w.slot >= 0 ? t * 128 + rr : (int64_t)(w.row0 + i) * A.heads + w.h * A.group + g;
            int64_t row4[4];
            float inv4[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                row4[x] = __shfl_sync(0xffffffffu, orow, (lane >> 2) + 8 * x);
                inv4[x] = __shfl_sync(0xffffffffu, inv, (lane >> 2) + 8 * x);
            }
            T *const dst = reinterpret_cast<T *>(A.out) + (lane & 3) * 8;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                uint32_t v[2][16];                                   // rows lane / 4 + 16 x (+ 8: the upper two of four)
                if (w.nk > 0) {
                    ap_tmem_ld_rows(t_o + c0, v[0]);
                    ap_tmem_ld_rows(t_o + c0 + (16u << 16), v[1]);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (row4[x] < 0) continue;
                    float y[8];                                      // (a row without keys: whatever v holds)
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = inv4[x] != 0.0f ? __uint_as_float(v[x >> 1][4 * (e >> 1) + 2 * (x & 1) + (e & 1)]) * inv4[x] : 0.0f;
                    if (w.slot < 0) {
                        T z[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) z[e] = from_f32<T>(y[e]);
                        *reinterpret_cast<uint4 *>(dst + row4[x] * D + c0) = *reinterpret_cast<const uint4 *>(z);
                    } else {
                        float *to = part + row4[x] * D + c0 + (lane & 3) * 8;
                        *reinterpret_cast<float4 *>(to) = make_float4(y[0], y[1], y[2], y[3]);
                        *reinterpret_cast<float4 *>(to + 4) = make_float4(y[4], y[5], y[6], y[7]);
                    }
                }
            }
            tc_fence_before();                                       // O has been read before the next item's P is announced
            if (w.slot >= 0) {
                if (live) *reinterpret_cast<float2 *>(part + TILES * 128 * D + 2 * orow) = make_float2(m - AP_LIFT, l);
            } else if (live && A.lse != nullptr) A.lse[orow] = l == 0.0f ? __int_as_float(0xff800000) : (m - AP_LIFT + __log2f(l)) * 0.69314718f;
        }
    }
#undef AP_WAIT
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) A.wide[blockIdx.x] = *wide;
    if (warp == AP_MMA) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
template <int D, int BS, typename T>
static int ap_launch(const Attn4Args &a, bool split, cudaStream_t st, int *grid_out) {
    using S = ApSmem<D, BS>;
    constexpr int smem = S::TOTAL;
    static_assert(smem <= 227 * 1024, "shared memory of the prompt kernel");
    static bool configured[64] = {};
    int dev = 0;
    MPSBNB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        if (!attn4_smem_at(dev, 1024)) return MPSBNB_ERR_UNSUPPORTED;
        MPSBNB_CUDA_TRY(cudaFuncSetAttribute(attn4_prompt_kernel<D, BS, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        cudaFuncAttributes at;
        MPSBNB_CUDA_TRY(cudaFuncGetAttributes(&at, attn4_prompt_kernel<D, BS, T>));
        if (at.numRegs != AP_REGS) return MPSBNB_ERR_UNSUPPORTED;    // the warpgroups' shares are made for this number
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    // no more blocks than there can be items: a sequence's last block of rows may be partly filled
    const int64_t most = a.kv.kv_heads * (((int64_t)a.sq.tokens * a.group) / (S::TILES * 128) + a.sq.batch);
    const int sms = sm_count();
    const int grid = split || most > sms ? sms : (int)most;
    *grid_out = grid;
    attn4_prompt_kernel<D, BS, T><<<grid, AP_THREADS, smem, st>>>(a, split);
    const int rc = check_launch();
    return rc != MPSBNB_OK || !split ? rc : attn4_combine<D, S::TILES * 128, ATTN4_JOIN_WARPS, T>(a, grid, st);
}

size_t attn4_prompt_ws(int head_dim) {
    const int rows = head_dim == 256 ? 128 : 256;
    return (size_t)sm_count() * (2 * rows * (head_dim + 2) * sizeof(float) + sizeof(Attn4Join));
}

int attn4_prompt(const Attn4Args &a, int head_dim, int blocksize, int dtype, bool split, cudaStream_t st, int *grid) {
#define AP_PICK(D, BS) return dtype == MPSBNB_F16 ? ap_launch<D, BS, __half>(a, split, st, grid) : ap_launch<D, BS, __nv_bfloat16>(a, split, st, grid)
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
