// Attention over the paged 4-bit cache for few query rows per sequence (single tokens, drafts) - and, row tile by row
// tile, for any number of them.  out = softmax(scale q K^T) V, K = code * absmax, V = code * absmax.
//
// Floor: HBM, for the cached bytes (head_dim / 2 + 2 head_dim / blocksize per token, head and side) are read once and
// the arithmetic per byte is small.  Bound: turning 4-bit codes into operands at that rate.  64 sequences of up to 16384 places
// (8 kv heads of 128, 8 query heads each: 545 MB) take 152 us, 3.6 TB/s, 0.55 of what a copy reaches; 57 % of the issue slots and 60 %
// of the load pipe are then in use (331 instructions and 64 look-ups a lane for 16 tokens; of 108 wavefronts of shared memory 18 are
// conflicts of the loads of codes, 64 bytes a row: tokens four apart for K, two for V), the tensor pipe at 22 %.  No unit is at its
// limit: most stalls are fixed latencies, with three warps a scheduler to hide them.  Tried for it: 8 warps a block (+20 %) and 16 (=) for
// 12; codes straight from global memory instead of the ring (+10 %); the next tile's scores under this one's values (=); all look-ups of
// a block before its products (=).  head_dim 256 with 16-row tiles spills 420 - 520 bytes a thread, the others next to nothing.
// Little work is bound by latency: 14 us for two launches, however short the sequences are (32 heads of 200 keys).
//
//  * Work is a list of (sequence, kv head, row tile, key tile), cut into equal runs, one per team of four warps,
//    whatever the sequences' lengths are: the lengths are read on the device, so a captured graph follows them.
//    A run that begins or ends inside a (sequence, head, row tile) leaves a partial result in the workspace, and
//    attn4_combine_kernel joins the partials.
//  * A key tile is one or two groups of the cache: a bulk copy each into the warp's own ring of stages.  No barrier between
//    warps while tiles stream; a warp waits on its own mbarriers only.
//  * S^T = K Q^T and O^T = V^T P^T with mma.m16n8k16: tokens (then channels) are the 16 rows and the query rows
//    the 8 columns, so a group of up to 8 heads wastes nothing of the tile.  (tcgen05 would want 128 rows and the
//    operands in shared memory: here they are made in registers.)  Codes become fp16 pairs by a 256-entry table
//    of byte -> (low nibble's value, high nibble's), held once per lane so that 32 look-ups never meet in a bank.
//    For V the pair has to run along tokens: the nibbles of two tokens' words are first brought into one byte.
//  * A block's absmax multiplies the fp32 score (K) or the probability (V), never a code: K enters the product
//    with the rounding of the 16 code values to fp16 only.
//  * Softmax: probabilities are 2^(x - m) with a reference m that follows the running maximum only when a score
//    exceeds it by 2^8: one vote per tile instead of a reduction, and fp32 sums lose nothing by it.  The weight
//    p * absmax goes to fp16 (off by 2^-11 at most, 2.1e-4 in the root mean square; a second fp16 for the rest would cost a third
//    more products and conversions): an output is off by 2.9e-4 - 3.6e-4 of its size, where its own rounding to fp16 makes 2.1e-4;
//    in bf16 nothing is to be seen of it.  absmax is taken times a power of two that brings a tile's to [2^-4, 2^7]; the same
//    vote sees when they leave that.  A tile that has more between its smallest and its largest takes a power of two for each row
//    and block, after that row's largest weight: what other rows see, or what has next to no weight, costs a row no bits.  (The
//    vote and the room in the instruction cache cost 1.5 - 3 %; a cache all of whose tiles are like that takes half as long again.)
//    bf16 queries are brought to fp16 by a power of two per row: exact, but for parts below 2^-24 of the row's largest.
#include <cmath>
#include <type_traits>

#include "attn4.cuh"

namespace mpsbnb {

using namespace sm100;

static __device__ int g_attn4_status = 0;

constexpr int AD_WARPS = 4;                                          // of a team: the warps that share a run of tiles
// What a (sequence, head, row tile) counts besides its tokens, in tokens: q, the joining of the warps
constexpr int AD_COST_TOKENS = 512;
// An absmax up to 1e-8 (as bf16 has it) is the quantiser's floor, or 0 in fp16: its block is nothing beside others.
constexpr uint32_t AD_ABOVE_FLOOR = 0x322c0001u;
constexpr uint32_t AD_LUT = 65536;                                   // shared-window address of the table
constexpr uint32_t AD_BASE = 1024;                                   // ... and of the dynamic shared memory

// A block has one table (256 entries of 256 bytes, the lower 128 of which are in use: lane l's copy at 4 l) on a 64 KB
// boundary, so that one byte permute makes a look-up's address.  It is too large for two blocks on an SM; instead a
// block holds TEAMS teams of four warps which do not wait on one another.
template <int D, int BS, int NT> struct AdSmem {
    static constexpr int WARPS = D * NT <= 128 ? 12 : 8, THREADS = WARPS * 32;   // 168 or 255 registers a thread
    static constexpr int TEAMS = WARPS / AD_WARPS;
    static constexpr int GROUP = 2 * kv4_half_bytes(D, BS);
    static constexpr int G = D == 256 ? 1 : 2;                       // groups of 16 tokens per tile
    static constexpr int TOK = 16 * G;                               // tokens per tile
    static constexpr int STAGE = G * GROUP, STAGES = D == 128 ? 2 : 3;   // of a warp's ring
    static constexpr int COST = AD_COST_TOKENS / TOK;
    static constexpr int RT = 8 * NT;
    static constexpr int RED_D = D == 256 ? 64 : D, RED_LD = RED_D + 2;   // channels, floats per row of a merge pass
    // window addresses: the rings of as many warps as fit before the table, the others and the rest behind it
    static constexpr int FIT = (AD_LUT - AD_BASE) / (STAGES * STAGE);
    static constexpr int WARPS0 = FIT < WARPS ? FIT : WARPS;
    static constexpr uint32_t RING0 = AD_BASE, RING1 = AD_LUT + 65536;
    static constexpr uint32_t RED = RING1 + (WARPS - WARPS0) * STAGES * STAGE;
    static constexpr uint32_t STAT = RED + WARPS * RT * RED_LD * 4;  // (maximum, sum) of every warp and row
    static constexpr uint32_t BAR = STAT + WARPS * RT * 8;
    static constexpr uint32_t REDO = BAR + WARPS * STAGES * 8 + 4, END = REDO + 12;   // (the word before it: abort flag)
    static constexpr int BYTES = END - AD_BASE;
    static_assert(BYTES <= 227 * 1024, "shared memory of the decode kernel");
    static_assert(GROUP % 16 == 0, "bulk copies go by 16 bytes");
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
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t ad_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// NB consecutive 16-bit absmax values as floats.  This and the loads of codes are volatile, which keeps them between the waits
// and releases of their stage, but clobber nothing: the look-ups may be scheduled around them.
template <typename T, int NB> __device__ __forceinline__ void ad_scales(uint32_t addr, float (&s)[NB]) {
    uint32_t w[(NB + 1) / 2];
    if constexpr (NB == 1) { uint16_t h; asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(addr)); w[0] = h; }
    else if constexpr (NB == 2) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
    else if constexpr (NB == 4) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    else asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        s[i] = to_f32<T>(*reinterpret_cast<const T *>(&h));
    }
}

// A sequence as this kernel walks it: rows = (new token, head of the group) pairs in tiles of RT rows, keys in tiles of TOK places.
struct AdSeq {
    int row0, n, len;                            // first row of q, new tokens, places
    int tlo, nt;                                 // first key tile and number of key tiles (one dead tile if there is no key)
    int rts;                                     // row tiles
    template <class S> __device__ __forceinline__ void get(const Attn4Args &a, int b) {
        a.sq.get(b, row0, n, len);
        if (n * a.group > a.rows_hi || n * a.group <= a.rows_lo) n = 0;
        if (a.redo) {
            uint32_t mask;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(mask) : "r"(S::REDO) : "memory");
            if (!(mask >> (b & 31) & 1u)) n = 0;
        }
        const int low = a.window > 0 ? max(0, len - n - a.window + 1) : 0;
        tlo = low / S::TOK;
        nt = n > 0 ? max((len + S::TOK - 1) / S::TOK - tlo, 1) : 0;
        rts = (n * a.group + S::RT - 1) / S::RT;
    }
    // units of work: key tiles, and COST more for each (head, row tile)
    template <class S> __device__ __forceinline__ int64_t units(const Attn4Args &a) const { return nt > 0 ? (int64_t)(nt + S::COST) * rts * a.kv.kv_heads : 0; }
};
template <class S> __device__ __forceinline__ int64_t ad_units(const Attn4Args &a, int b) {
    if (b >= a.sq.batch) return 0;
    AdSeq s;
    s.get<S>(a, b);
    return s.units<S>(a);
}
// sum over the lanes up to this one
__device__ __forceinline__ int64_t ad_scan(int64_t x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += up;
    }
    return x;
}
// n / d for n >= 0, d > 0, in 32 bits where they do
__device__ __forceinline__ int64_t ad_div(int64_t n, int64_t d) {
    return n < 0x7fffffffll && d < 0x7fffffffll ? (int64_t)((uint32_t)n / (uint32_t)d) : n / d;
}

// A walk over the pieces (runs of key tiles of one sequence, head and row tile) of a team's run.  Runs are cut in units: a
// (sequence, head, row tile) counts COST units at its beginning and then its key tiles.
template <class S> struct AdPiece {
    AdSeq s;
    int b, h, r;                                 // sequence, kv head, row tile
    int a, e;                                    // key tiles of the piece, relative to s.tlo
    int64_t left;                                // units of the run after this piece

    // first piece of the run [t0, t1) of the whole list (false: the run holds none of its tiles); whole warp.  (The ends of the
    // walk are checked: lengths that change under a running kernel must not lead it outside.)
    // w, inc: units of sequence `lane`, and of the sequences up to it
    __device__ __forceinline__ bool start(const Attn4Args &A, int64_t w, int64_t inc, int64_t t0, int64_t t1) {
        const int lane = threadIdx.x & 31;
        int64_t base = 0;
        for (int b0 = 0;; b0 += 32) {
            if (b0 >= A.sq.batch) return false;
            if (b0 > 0) {
                w = ad_units<S>(A, b0 + lane);
                inc = ad_scan(w);
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
        s.get<S>(A, b);
        const int64_t off = t0 - base;
        const int units = s.nt + S::COST, sub = (int)ad_div(off, units);
        h = sub / s.rts;
        r = sub - h * s.rts;
        left = t1 - t0;
        take(A, (int)(off - (int64_t)sub * units));
        return e > 0 || next(A);
    }
    // the piece that begins `from` units into its (sequence, head, row tile)
    __device__ __forceinline__ void take(const Attn4Args &A, int from) {
        int to = (int)min((int64_t)(s.nt + S::COST), from + left);
        left -= to - from;
        if (A.redo) to = from == 0 ? s.nt + S::COST : 0;             // nothing is cut: whole ones, in the runs that they begin in
        a = max(0, from - S::COST);
        e = max(0, to - S::COST);
    }
    // next piece; false when the run is done
    __device__ __forceinline__ bool next(const Attn4Args &A) {
        do {
            if (left == 0) return false;
            if (++r == s.rts) {
                r = 0;
                if (++h == A.kv.kv_heads) {
                    h = 0;
                    do {
                        if (++b >= A.sq.batch) return false;
                        s.get<S>(A, b);
                    } while (s.nt == 0);
                }
            }
            take(A, 0);
        } while (e == 0);
        return true;
    }
};

// Units per team: equal, and no fewer than give each warp two tiles and then some.  (What little work there is is best spread
// thin: 32 heads of 200 keys take 15.4 us so, 17.4 with a piece's cost and a tile for each warp, 19.5 with four tiles.)
__device__ __forceinline__ int64_t ad_per(int64_t total, int teams, int cost) { return max(ad_div(total + teams - 1, teams), (int64_t)(cost / 4 + 2 * AD_WARPS)); }

template <int D, int BS, int NT, typename T>
__global__ void __launch_bounds__((AdSmem<D, BS, NT>::THREADS), 1)
attn4_decode_kernel(const __grid_constant__ Attn4Args A) {
    using S = AdSmem<D, BS, NT>;
    using Piece = AdPiece<S>;
    constexpr int NB = D / BS, MT = D / 16, MB = BS / 16, RT = S::RT, G = S::G;   // MB: k steps, and channel tiles, per block
    constexpr int HALF = kv4_half_bytes(D, BS), SOFF = KV4_GROUP * (D / 2);
    extern __shared__ __align__(128) unsigned char smem[];
    if (A.redo) pdl_grid_dependency_wait();                          // (before any return: this kernel's end means the ends of those before)
    if (smem_u32(smem) != AD_BASE) {                                 // the layout counts on it
        if (threadIdx.x == 0) atomicExch(&g_attn4_status, 403);      // (and nothing to join)
        if (!A.redo && threadIdx.x < S::TEAMS) attn4_join<D, RT>(A.ws, gridDim.x * S::TEAMS)[threadIdx.x * gridDim.x + blockIdx.x].n = 0;
        return;
    }
    const int cta_warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int in_team = cta_warp / AD_WARPS, warp = cta_warp % AD_WARPS;
    const int teams = gridDim.x * S::TEAMS, team = in_team * gridDim.x + blockIdx.x;   // little work spreads over the SMs
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + (S::END - 16 - AD_BASE));
    if (A.redo) {                                                    // (mostly there is nothing to do)
        if (__syncthreads_or(threadIdx.x < A.wide_n && __ldcg(A.wide + threadIdx.x) != 0) == 0) return;
        uint32_t mask = 0;
        for (int i = lane; i < A.wide_n; i += 32) mask |= __ldcg(A.wide + i);
        mask = __reduce_or_sync(0xffffffffu, mask);
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(S::REDO), "r"(mask) : "memory");
        __syncwarp();
    }
    // little work is a chain of small loads: those of the lengths, and of the page table into L2, are under way while the table is made
    const int64_t units = ad_units<S>(A, lane);
    if (cta_warp == 0 && lane < A.sq.batch && A.sq.capacity > 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(A.sq.table + (int64_t)lane * A.sq.table_ld));
    pdl_launch_dependents();

    // ------------------------------------------------------------ table, barriers
    if (threadIdx.x < 256) {
        // a byte to a thread: its pair 32 times, 16 bytes at a time and each lane beginning elsewhere (no two in a bank)
        const uint32_t pair = ad_half2(A.code[threadIdx.x & 15], A.code[threadIdx.x >> 4]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(AD_LUT + threadIdx.x * 256 + ((i + lane) & 7) * 16), "r"(pair) : "memory");
    }
    if (threadIdx.x < S::WARPS * S::STAGES) mbar_init(S::BAR + 8 * threadIdx.x, G);
    if (threadIdx.x == 0) *abort_flag = 0;
    fence_mbar_init();

    // ------------------------------------------------------------ my team's run
    const int64_t inc = ad_scan(units);
    int64_t total = __shfl_sync(0xffffffffu, inc, 31);
    if (A.sq.batch > 32) {
        int64_t more = 0;
        for (int b = 32 + lane; b < A.sq.batch; b += 32) more += ad_units<S>(A, b);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) more += __shfl_xor_sync(0xffffffffu, more, o);
        total += more;
    }
    const int64_t per = ad_per(total, teams, S::COST), t0 = min(total, team * per), t1 = min(total, t0 + per);
    // what the teams leave for attn4_combine_kernel (a team's thread 0 writes both)
    Attn4Join *join = attn4_join<D, RT>(A.ws, teams) + team;
    if (!A.redo && warp == 0 && lane == 0) join->n = 0;
    Piece in;                                                        // piece the next copy belongs to
    const bool some = t0 < t1 && in.start(A, units, inc, t0, t1);
    __syncthreads();
    if (!some) return;                                               // whole team; no barrier of the block follows
    Piece cur = in;                                                  // piece being worked on
    auto team_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(in_team + 1), "n"(AD_WARPS * 32) : "memory"); };
    const uint32_t lut = AD_LUT + lane * 4;
    const uint32_t ring = cta_warp < S::WARPS0 ? S::RING0 + cta_warp * (S::STAGES * S::STAGE) : S::RING1 + (cta_warp - S::WARPS0) * (S::STAGES * S::STAGE);
    const uint32_t bars = S::BAR + cta_warp * S::STAGES * 8;
    const bool negate = A.scale_log2 < 0.0f;                         // a negative scale goes into q: maxima stay maxima

    // ------------------------------------------------------------ producer side: this warp's tiles, in order
    // tiles of a piece that this warp takes (every fourth; none of an empty sequence's dead tile)
    auto tiles_of = [&](const Piece &p) {
        const int end = min(p.e, (p.s.len + S::TOK - 1) / S::TOK - p.s.tlo);
        return max(0, (end - p.a - warp + AD_WARPS - 1) / AD_WARPS);
    };
    constexpr int BATCH = 32 / G;                                    // tiles whose addresses the lanes hold, a group each
    int in_k = 0, in_n = tiles_of(in);                               // next of how many
    uint64_t in_addr = 0;                                            // where my group lies; 0: nowhere
    uint32_t in_bad = 0;                                             // lanes whose group is in a page outside the cache
    uint32_t put = 0;                                                // next stage to fill
    bool in_more = true;
    auto issue = [&]() {                                             // whole warp
        while (in_k == in_n) {
            if (!in_more) return;
            in_more = in.next(A);
            in_k = 0;
            in_n = in_more ? tiles_of(in) : 0;
        }
        const int at = in_k % BATCH;
        if (at == 0) {
            in_addr = 0;
            bool bad = false;
            const int place = (in.s.tlo + in.a + warp + (in_k + lane / G) * AD_WARPS) * S::TOK + (lane % G) * 16;
            if (in_k + lane / G < in_n && place < in.s.len) {
                const int page = __ldg(A.sq.table + (int64_t)in.b * A.sq.table_ld + (place >> A.kv.page_shift));
                bad = page < 0 || page >= A.kv.num_pages;
                if (!bad) in_addr = reinterpret_cast<uint64_t>(A.kv.group(page, in.h, place));
            }
            in_bad = __ballot_sync(0xffffffffu, bad);
        }
        const uint32_t full = bars + 8 * put, dst = ring + put * S::STAGE;
        if (in_bad >> (at * G) & ((1u << G) - 1u)) {
            // a page outside the cache: its keys' absmax is NaN, and so is every row that sees them; its values' is 0, not what lies there
#pragma unroll
            for (int x = 0; x < G; ++x)
                if (in_bad >> (at * G + x) & 1u)
                    for (int i = lane; i < KV4_GROUP * NB; i += 32) {
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + x * S::GROUP + SOFF + 2 * i), "h"((uint16_t)0x7fff) : "memory");
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + x * S::GROUP + HALF + SOFF + 2 * i), "h"((uint16_t)0) : "memory");
                    }
            if (lane == 0) atomicExch(&g_attn4_status, KV4_BAD_PAGE);
            __syncwarp();
        }
        if (lane / G == at) {                                        // each of the tile's lanes fetches its own group
            if (in_addr != 0) {
                mbar_arrive_expect_tx(full, S::GROUP);
                bulk_load_1d(dst + (lane % G) * S::GROUP, reinterpret_cast<const void *>(in_addr), S::GROUP, full);
            } else {
                mbar_arrive(full);
            }
        }
        put = put == S::STAGES - 1 ? 0 : put + 1;
        ++in_k;
    };
#pragma unroll 1
    for (int i = 0; i < S::STAGES; ++i) issue();

    // ------------------------------------------------------------ consumer side
    // A-operand row r of a group is token r / 2 (even r) or r / 2 + 4 (odd r), + 8 for rows 8 .. 15: the k index of P^T
    // below then gives a lane the tokens c, c + 4, c + 8, c + 12
    const int tok = (g >> 1) + 4 * (g & 1);
    uint32_t got = 0, phase = 0;                                     // next stage to read, its barrier's parity
    bool first_piece = true;
    do {
        const AdSeq &sq = cur.s;
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
        bool far = false;                                            // some column's reference is

        int place0 = (sq.tlo + cur.a + warp) * S::TOK;
#pragma unroll 1
        for (int left = tiles_of(cur); left > 0; --left, place0 += AD_WARPS * S::TOK) {
            if (!mbar_wait(bars + 8 * got, phase, abort_flag)) { atomicExch(&g_attn4_status, 402); *abort_flag = 1; }
            const uint32_t kb = ring + got * S::STAGE;
            // scores: s[x][nt][0..1] token tok of group x, columns 2c and 2c + 1; s[x][nt][2..3] token tok + 8
            float s[G][NT][4];
#pragma unroll
            for (int x = 0; x < G; ++x) {
                const uint32_t kx = kb + x * S::GROUP;
                float sc0[NB], sc1[NB];
                ad_scales<T, NB>(kx + SOFF + tok * NB * 2, sc0);
                ad_scales<T, NB>(kx + SOFF + (tok + 8) * NB * 2, sc1);
#pragma unroll
                for (int blk = 0; blk < NB; ++blk) {
                    uint32_t w0[MB / 2], w1[MB / 2];
                    const uint32_t ka = kx + tok * (D / 2) + blk * (BS / 2) + c * (BS / 8);
                    if constexpr (BS == 64) {
                        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w0[0]), "=r"(w0[1]) : "r"(ka));
                        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w1[0]), "=r"(w1[1]) : "r"(ka + 8 * (D / 2)));
                    } else {
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w0[0]) : "r"(ka));
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w1[0]) : "r"(ka + 8 * (D / 2)));
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
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float sc = j < 2 ? sc0[blk] : sc1[blk];
                            s[x][nt][j] = blk == 0 ? sc * acc[nt][j] : fmaf(sc, acc[nt][j], s[x][nt][j]);
                        }
                }
            }
            // absmax of the values, token tok (+ 8) of group x
            float sv[G][2][NB], sm = 0.0f, sn = __int_as_float(0x7f800000);
#pragma unroll
            for (int x = 0; x < G; ++x) {
                ad_scales<T, NB>(kb + x * S::GROUP + HALF + SOFF + tok * NB * 2, sv[x][0]);
                ad_scales<T, NB>(kb + x * S::GROUP + HALF + SOFF + (tok + 8) * NB * 2, sv[x][1]);
            }
            uint32_t seen = 0xffffffffu;                             // bit (x * NT + nt) * 4 + j
            if (place0 < full_lo || place0 + S::TOK > full_hi) {     // some row does not see some key (full_hi <= len)
                seen = 0;
#pragma unroll
                for (int x = 0; x < G; ++x) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int place = place0 + 16 * x + tok + 8 * (j >> 1);
                            if (place < lim[nt][j & 1] && place >= low[nt][j & 1]) seen |= 1u << ((x * NT + nt) * 4 + j);
                            else s[x][nt][j] = __int_as_float(0xff800000);
                        }
                    // whatever lies in a place that no row sees
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int place = place0 + 16 * x + tok + 8 * y;
                        if (place < any_lo || place >= any_hi) {
#pragma unroll
                            for (int blk = 0; blk < NB; ++blk) sv[x][y][blk] = 0.0f;
                        }
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < G; ++x)
#pragma unroll
                for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        sm = fmaxf(sm, sv[x][y][blk]);
                        sn = fminf(sn, sv[x][y][blk]);
                    }
            float p[G][NT][4], top = -1.0f;
#pragma unroll
            for (int x = 0; x < G; ++x)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        p[x][nt][j] = fmaf(s[x][nt][j], f[nt][j & 1], -m[nt][j & 1]);
                        top = fmaxf(top, p[x][nt][j]);
                    }
            // lane (g, c): channels blk * BS + g * (BS / 8) + 0 .. BS / 8 - 1 of the tokens c, c + 4, c + 8, c + 12 of group x, those
            // of two tokens in a byte: ev the even channels, od the odd ones
            auto codes_of = [&](int x, int blk, uint32_t (&ev)[2], uint32_t (&od)[2]) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t va = kb + x * S::GROUP + HALF + (c + 4 * i) * (D / 2) + blk * (BS / 2) + g * (BS / 16);
                    if constexpr (BS == 64) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(va));
                    else { uint16_t h; asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(va)); w[i] = h; }
                }
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    ev[y] = (w[2 * y] & 0x0F0F0F0Fu) | ((w[2 * y + 1] << 4) & 0xF0F0F0F0u);
                    od[y] = ((w[2 * y] >> 4) & 0x0F0F0F0Fu) | (w[2 * y + 1] & 0xF0F0F0F0u);
                }
            };
            auto weights = [&](const float (&pr)[4], int x, int blk, int nt, float (&wt)[4]) {
#pragma unroll
                for (int j = 0; j < 4; ++j) wt[j] = pr[j] * (sv[x][j >> 1][blk] * up);
                if (seen != 0xffffffffu) {                           // a value that is not finite is no matter of rows that do not see it
#pragma unroll
                    for (int j = 0; j < 4; ++j) if (!(seen >> ((x * NT + nt) * 4 + j) & 1u)) wt[j] = 0.0f;
                }
            };
            // p stays under 2^8 and absmax * up in [2^-4, 2^7]: their product is at home in fp16
            auto least = [&]() { return __int_as_float((250 << 23) - __float_as_int(up)); };   // 2^-4 / up
            const bool high = top > 8.0f || sm * up > 128.0f || far;
            if (__any_sync(0xffffffffu, high || sn < least())) {
                uint32_t sl = 0xffffffffu;                           // the least above the floor, as bits from there on
#pragma unroll
                for (int x = 0; x < G; ++x)
#pragma unroll
                    for (int blk = 0; blk < NB; ++blk)
#pragma unroll
                        for (int y = 0; y < 2; ++y) sl = min(sl, __float_as_uint(sv[x][y][blk]) - AD_ABOVE_FLOOR);
                sl = __reduce_min_sync(0xffffffffu, sl);
                auto low = [&]() { return sl < (uint32_t)max(0, (int)(__float_as_uint(least()) - AD_ABOVE_FLOOR)); };
                if (__any_sync(0xffffffffu, high || low())) {
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) sm = fmaxf(sm, __shfl_xor_sync(0xffffffffu, sm, d));
                    float ku = 1.0f;
                    // the largest comes to [16, 32); up is held in [2^-40, 2^100], where the sums are in no danger
                    const float un = __int_as_float(max(87, min(227, 258 - (int)(__float_as_uint(fminf(sm, 3.4e38f)) >> 23))) << 23);
                    if (sm * up > 128.0f) {
                        ku = un * __frcp_rn(up);                     // (0 where the difference leaves fp32)
                        up = un;
                    } else if (low() && un > up) {                   // up again, if the sums allow it
                        float most = 0.0f;
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(o[i][nt][j]));
#pragma unroll
                        for (int d = 1; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                        const float more = un * __frcp_rn(up);
                        if (most * more < 0x1p100f) { ku = more; up = un; }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float mx = fmaxf(s[0][nt][j], s[0][nt][j + 2]);
                            if (G == 2) mx = fmaxf(mx, fmaxf(s[G - 1][nt][j], s[G - 1][nt][j + 2]));
                            mx *= f[nt][j];
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                            const float mn = mx > m[nt][j] + (fabsf(m[nt][j]) < ATTN4_FAR ? 8.0f : 0.0f) ? mx : m[nt][j], k = ex2(m[nt][j] - mn);
                            const bool off = fabsf(mn) >= ATTN4_FAR && mn != ATTN4_NONE;
                            far = far || off;
                            m[nt][j] = mn;
                            l[nt][j] *= k;
#pragma unroll
                            for (int i = 0; i < MT; ++i) { o[i][nt][j] *= k * ku; o[i][nt][j + 2] *= k * ku; }
#pragma unroll
                            for (int x = 0; x < G; ++x) {
                                p[x][nt][j] = off ? __fmul_rn(s[x][nt][j], f[nt][j]) - mn : fmaf(s[x][nt][j], f[nt][j], -mn);
                                p[x][nt][j + 2] = off ? __fmul_rn(s[x][nt][j + 2], f[nt][j]) - mn : fmaf(s[x][nt][j + 2], f[nt][j], -mn);
                            }
                        }
                    if (sm * up > 128.0f || low()) {
                        // The tile's absmax do not fit in there: each column's largest weight of a block to [16, 32), the products
                        // apart and back into up's unit.  To what follows the tile's values are zeros.
#pragma unroll
                        for (int blk = 0; blk < NB; ++blk) {
                            uint32_t b0[G][NT], b1[G][NT], ev[G][2], od[G][2];
                            float back[NT][2];
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                float wt[G][4], mul[2];
#pragma unroll
                                for (int x = 0; x < G; ++x) {
                                    const float pr[4] = {ex2(p[x][nt][0]), ex2(p[x][nt][1]), ex2(p[x][nt][2]), ex2(p[x][nt][3])};
                                    weights(pr, x, blk, nt, wt[x]);
                                }
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    float wm = fmaxf(fmaxf(wt[0][j], wt[0][j + 2]), fmaxf(wt[G - 1][j], wt[G - 1][j + 2]));
#pragma unroll
                                    for (int d = 4; d < 32; d <<= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, d));
                                    const int e = max(5, min(250, (int)(__float_as_uint(wm) >> 23)));
                                    mul[j] = __int_as_float((258 - e) << 23);            // 2^(131 - e)
                                    back[nt][j] = __int_as_float((e - 4) << 23);         // 2^(e - 131)
                                }
#pragma unroll
                                for (int x = 0; x < G; ++x) {
                                    b0[x][nt] = ad_transpose(ad_half2(wt[x][0] * mul[0], wt[x][1] * mul[1]));
                                    b1[x][nt] = ad_transpose(ad_half2(wt[x][2] * mul[0], wt[x][3] * mul[1]));
                                }
                            }
#pragma unroll
                            for (int x = 0; x < G; ++x) codes_of(x, blk, ev[x], od[x]);
#pragma unroll
                            for (int j = 0; j < MB; ++j) {
                                float t[NT][4];
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int i = 0; i < 4; ++i) t[nt][i] = 0.0f;
#pragma unroll
                                for (int x = 0; x < G; ++x) {
                                    const uint32_t a0 = ad_lut(lut, ev[x][0], j), a1 = ad_lut(lut, od[x][0], j), a2 = ad_lut(lut, ev[x][1], j), a3 = ad_lut(lut, od[x][1], j);
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt) ad_mma(t[nt], a0, a1, a2, a3, b0[x][nt], b1[x][nt]);
                                }
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int i = 0; i < 4; ++i) o[blk * MB + j][nt][i] = fmaf(t[nt][i], back[nt][i & 1], o[blk * MB + j][nt][i]);
                            }
                        }
#pragma unroll
                        for (int x = 0; x < G; ++x)
#pragma unroll
                            for (int blk = 0; blk < NB; ++blk) sv[x][0][blk] = sv[x][1][blk] = 0.0f;
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < G; ++x)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        p[x][nt][j] = ex2(p[x][nt][j]);
                        l[nt][j & 1] += p[x][nt][j];
                    }
            // O^T += V^T P^T
#pragma unroll
            for (int x = 0; x < G; ++x)
#pragma unroll
                for (int blk = 0; blk < NB; ++blk) {
                    uint32_t b0[NT], b1[NT], ev[2], od[2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float wt[4];
                        weights(p[x][nt], x, blk, nt, wt);
                        b0[nt] = ad_transpose(ad_half2(wt[0], wt[1]));
                        b1[nt] = ad_transpose(ad_half2(wt[2], wt[3]));
                    }
                    codes_of(x, blk, ev, od);
#pragma unroll
                    for (int j = 0; j < MB; ++j) {
                        const uint32_t a0 = ad_lut(lut, ev[0], j), a1 = ad_lut(lut, od[0], j), a2 = ad_lut(lut, ev[1], j), a3 = ad_lut(lut, od[1], j);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) ad_mma(o[blk * MB + j][nt], a0, a1, a2, a3, b0[nt], b1[nt]);
                    }
                }
            if (++got == S::STAGES) { got = 0; phase ^= 1; }
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
                const float k = ex2(m[nt][j] - M) * (__frcp_rn(up) * (attn4_code_unscale(A.quant_type) * ATTN4_SUM));
#pragma unroll
                for (int i = 0; i < MT; ++i) { o[i][nt][j] *= k; o[i][nt][j + 2] *= k; }
            }
        const bool whole = cur.a == 0 && cur.e == sq.nt;
        float *part = attn4_partial<D, RT>(A.ws, team, first_piece ? 0 : 1);
        if (cur.a == 0 && !whole && warp == 0 && lane == 0) {
            join->n = 1 + (int)((sq.nt - cur.e + per - 1) / per);
            join->slot = first_piece ? 0 : 1;
            join->row0 = sq.row0; join->rows = sq.n * A.group; join->r = cur.r; join->h = cur.h;
        }
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += S::RED_D) {                   // a pass is all channels, or 64 of 256
#pragma unroll
            for (int mt = d0 / 16; mt < (d0 + S::RED_D) / 16; ++mt) {
                const int d = mt / MB * BS + g * (BS / 8) + 2 * (mt % MB) - d0;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        *reinterpret_cast<float2 *>(red + (warp * RT + nt * 8 + 2 * c + j) * S::RED_LD + d) = make_float2(o[mt][nt][j], o[mt][nt][j + 2]);
            }
            team_sync();
            constexpr int PAIRS = S::RED_D / 2;
#pragma unroll
            for (int x = warp * 32 + lane; x < RT * PAIRS; x += AD_WARPS * 32) {
                const int row = x / PAIRS, d = 2 * (x % PAIRS), R = cur.r * RT + row, i = R / A.group;
                if (i >= sq.n) continue;
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
                    const float inv = L == 0.0f ? 0.0f : __fdividef(1.0f / ATTN4_SUM, L);
                    const int64_t orow = (int64_t)(sq.row0 + i) * A.heads + cur.h * A.group + (R - i * A.group);
                    T pr[2] = {from_f32<T>(v.x * inv), from_f32<T>(v.y * inv)};
                    *reinterpret_cast<uint32_t *>(reinterpret_cast<T *>(A.out) + orow * D + d0 + d) = *reinterpret_cast<const uint32_t *>(pr);
                    if (A.lse != nullptr && d0 == 0 && d == 0) A.lse[orow] = L == 0.0f ? __int_as_float(0xff800000) : (M + __log2f(L)) * 0.69314718f;
                } else {
                    *reinterpret_cast<float2 *>(part + row * D + d0 + d) = v;
                    if (d0 == 0 && d == 0) *reinterpret_cast<float2 *>(part + RT * D + 2 * row) = make_float2(M, L);
                }
            }
            team_sync();                                             // red (and, at the end, stat) may be written again
        }
        first_piece = false;
    } while (cur.next(A));
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
// The longest sequence's new tokens, for the choices below: what the caller says, but no more than is left when every other has one.
// (A caller that does not know says the number of all rows; single tokens are still seen for what they are.)
static int64_t ad_longest(const mpsbnb_kv4_seqs *s) {
    if (s->cu_seqlens == nullptr) return s->new_tokens;
    const int64_t most = s->tokens - (s->batch - 1) > 1 ? s->tokens - (s->batch - 1) : 1;
    return s->new_tokens < most ? s->new_tokens : most;
}
// 16 rows per tile where 8 do not hold a sequence's rows: the keys are then expanded half as often
static int ad_nt(const mpsbnb_kv4_seqs *s, int group) { return ad_longest(s) * group > 8 ? 2 : 1; }

// The tensor-core kernel of attn4_prompt.cu instead?  A key tile costs it the same whether its rows are 16 or 256: 2.0, 2.4, 3.3 us
// per 128 keys and block of rows on an SM (head_dim 64, 128, 256).  The kernel here spreads any amount of work over the whole card,
// at 0.42, 0.70, 1.83 ns per 16 rows x 16 keys, and begins and ends sooner, by 15, 20, 6 us.  So prompts go there when
// keys * (16-row tiles - 4.7, 2.9, 1.5 * blocks of rows) is above 570, 450, 50 thousand.  The keys are those that the table has room
// for: what the lengths are is known on the device alone.  (Measured for 1 - 8 sequences, 1 and 8 heads, 20 - 4096 rows a head and
// 1024 - 32768 keys.  8 heads, head_dim 128, here and there, us: 8192 keys of 64 rows 32 and 42, 256 rows 71 and 50, 1024 rows 210
// and 71; 1024 keys of 256 rows 28 and 46, 4096 rows 153 and 50.)
// Few blocks of rows (under AD_SPLIT rounds over the card) share out the keys as well; of many, a round begun counts as a whole one.
constexpr int AD_SPLIT = 2;
enum AdKind { AD_TOKENS, AD_PROMPTS, AD_PROMPTS_SPLIT };
static bool ad_split(const mpsbnb_kv4_cache *c, const mpsbnb_kv4_seqs *s, int group) {
    const int64_t block = c->head_dim == 256 ? 128 : 256;
    // (every block of the card looks through the (sequence, block of rows) pairs, 32 at a time)
    return (int64_t)s->batch * c->kv_heads * ((ad_longest(s) * group + block - 1) / block) <= AD_SPLIT * (int64_t)sm_count();
}
static AdKind ad_kind(const mpsbnb_kv4_cache *c, const mpsbnb_kv4_seqs *s, int group, int window) {
    const int64_t rows = (s->tokens * group + s->batch - 1) / s->batch;   // of a sequence and head, on average
    const int64_t lists = (int64_t)s->batch * c->kv_heads, block = c->head_dim == 256 ? 128 : 256, sms = sm_count();
    const int64_t blocks = lists * ((rows + block - 1) / block), tiles = lists * ((rows + 15) / 16);
    const bool split = ad_split(c, s, group);
    double keys = (double)s->table_width * c->page_size;
    if (window > 0 && keys > (double)window + ad_longest(s)) keys = (double)window + ad_longest(s);
    const int at = c->head_dim == 64 ? 0 : c->head_dim == 128 ? 1 : 2;
    const double meet[3] = {4.7, 2.9, 1.5}, sooner[3] = {570e3, 450e3, 50e3};
    if (rows <= 16 || keys * (tiles - meet[at] * (split ? blocks : (blocks + sms - 1) / sms * sms)) <= sooner[at]) return AD_TOKENS;
    return split ? AD_PROMPTS_SPLIT : AD_PROMPTS;
}

// Prompts among single tokens, as a server batches them: both kernels, each for its sequences.  It may be so where the longest has
// four times the average's rows and alone would go to the prompt kernel.  (256 sequences over 4096 keys, one with 2048 new tokens, 32
// heads on 8: 463 us; by the prompt kernel alone 1170, as two calls 156 and 276: one after the other, nothing overlaps.)
static bool ad_mixed(const mpsbnb_kv4_cache *c, const mpsbnb_kv4_seqs *s, int group, int window) {
    if (s->cu_seqlens == nullptr || 4 * s->tokens > (int64_t)s->batch * ad_longest(s)) return false;
    mpsbnb_kv4_seqs one = *s;
    one.batch = 1; one.new_tokens = (int)ad_longest(s); one.tokens = one.new_tokens;
    return ad_kind(c, &one, group, window) != AD_TOKENS;
}
// rows a head up to which a sequence of a mixed call counts as single tokens: the kernels' times per key meet at 4.7, 2.9, 1.5 tiles of
// 16 rows (above), taken up to whole tiles
static int ad_few_rows(int D) { return D == 64 ? 80 : D == 128 ? 48 : 32; }

// what a call runs: both kernels (mixed) or one; how the prompt kernel does; 8-row tiles of single tokens
struct AdPlan { bool mixed; AdKind prompts; int nt; };
static AdPlan ad_plan(const mpsbnb_kv4_cache *c, const mpsbnb_kv4_seqs *s, int group, int window) {
    if (ad_mixed(c, s, group, window)) return {true, ad_split(c, s, group) ? AD_PROMPTS_SPLIT : AD_PROMPTS, group > 8 ? 2 : 1};
    return {false, ad_kind(c, s, group, window), ad_nt(s, group)};
}

static int ad_teams(int D, int NT) { return sm_count() * ((D * NT <= 128 ? 12 : 8) / AD_WARPS); }

template <int D, int BS, int NT, typename T>
static int ad_launch(const Attn4Args &a, cudaStream_t st) {
    using S = AdSmem<D, BS, NT>;
    static bool configured[64] = {};
    int dev = 0;
    MPSBNB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        if (!attn4_smem_at(dev, AD_BASE)) return MPSBNB_ERR_UNSUPPORTED;   // the layout counts on it
        MPSBNB_CUDA_TRY(cudaFuncSetAttribute(attn4_decode_kernel<D, BS, NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const int teams = ad_teams(D, NT);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(teams / S::TEAMS);
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::BYTES;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = a.redo ? 1 : 0;
    MPSBNB_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn4_decode_kernel<D, BS, NT, T>, a));
    int rc = check_launch();
    if (rc != MPSBNB_OK || a.redo) return rc;
    return attn4_combine<D, S::RT, 1, T>(a, teams, st);
}

template <int D, int BS>
static int ad_launch_t(const Attn4Args &a, int dtype, int nt, cudaStream_t st) {
    if (dtype == MPSBNB_F16) return nt == 1 ? ad_launch<D, BS, 1, __half>(a, st) : ad_launch<D, BS, 2, __half>(a, st);
    return nt == 1 ? ad_launch<D, BS, 1, __nv_bfloat16>(a, st) : ad_launch<D, BS, 2, __nv_bfloat16>(a, st);
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

// bytes of workspace: partial results of the kernel here, then - where prompts may go to the other one - a word for each of its blocks
// and its partial results
static size_t ad_wide_ws() { return ((size_t)sm_count() * sizeof(uint32_t) + 15) & ~(size_t)15; }
static size_t ad_tokens_ws(int D, int nt) {
    return ((size_t)ad_teams(D, nt) * (2 * (8 * nt) * (D + 2) * sizeof(float) + sizeof(Attn4Join)) + 15) & ~(size_t)15;
}

static size_t ad_tokens_ws(const mpsbnb_kv4_cache *c, const mpsbnb_kv4_seqs *s, int group) {
    const size_t any = ad_tokens_ws(c->head_dim, ad_nt(s, group)), mixed = ad_tokens_ws(c->head_dim, group > 8 ? 2 : 1);
    return any > mixed ? any : mixed;
}
static int ad_run(const Attn4Args &a, const mpsbnb_kv4_cache *c, int nt, cudaStream_t st) {
    if (c->blocksize == 32) {
        if (c->head_dim == 64) return ad_launch_t<64, 32>(a, c->dtype, nt, st);
        if (c->head_dim == 128) return ad_launch_t<128, 32>(a, c->dtype, nt, st);
        return ad_launch_t<256, 32>(a, c->dtype, nt, st);
    }
    if (c->head_dim == 64) return ad_launch_t<64, 64>(a, c->dtype, nt, st);
    if (c->head_dim == 128) return ad_launch_t<128, 64>(a, c->dtype, nt, st);
    return ad_launch_t<256, 64>(a, c->dtype, nt, st);
}
// the prompt kernel, and behind it the one here for what that does not take (16 rows per tile: there are many)
static int ad_prompt(Attn4Args a, const mpsbnb_kv4_cache *c, bool split, cudaStream_t st) {
    float *const ws = a.ws;
    a.ws = reinterpret_cast<float *>(reinterpret_cast<char *>(a.wide) + ad_wide_ws());
    const int rc = attn4_prompt(a, c->head_dim, c->blocksize, c->dtype, split, st, &a.wide_n);
    if (rc != MPSBNB_OK) return rc;
    a.ws = ws;
    a.redo = 1;
    return ad_run(a, c, 2, st);
}

extern "C" size_t mpsbnb_attention_4bit_workspace_bytes(const mpsbnb_kv4_cache *cache, const mpsbnb_kv4_seqs *seqs, int heads) {
    if (kv4_check_cache(cache, 0) != MPSBNB_OK || kv4_check_seqs(seqs, cache) != MPSBNB_OK) return 0;
    if (heads <= 0 || heads % cache->kv_heads != 0 || seqs->batch == 0 || seqs->tokens == 0) return 0;
    const int group = heads / cache->kv_heads;
    // (a window, not known here, may take the prompt kernel out, not bring it in)
    const AdKind kind = ad_kind(cache, seqs, group, 0);
    const bool mixed = ad_mixed(cache, seqs, group, 0);
    return ad_tokens_ws(cache, seqs, group) + (kind != AD_TOKENS || mixed ? ad_wide_ws() : 0) +
           (kind == AD_PROMPTS_SPLIT || mixed ? attn4_prompt_ws(cache->head_dim) : 0);
}

extern "C" int mpsbnb_attention_4bit(const mpsbnb_kv4_cache *cache, int layer, const mpsbnb_kv4_seqs *seqs, const void *q,
                                     int64_t q_token_stride, int64_t q_head_stride, int heads, int causal, int window, float scale,
                                     void *out, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = kv4_check_cache(cache, layer);
    if (rc == MPSBNB_OK) rc = kv4_check_seqs(seqs, cache);
    if (rc != MPSBNB_OK) return rc;
    if (heads <= 0 || heads % cache->kv_heads != 0 || window < 0 || (window > 0 && !causal) || !(fabsf(scale) < INFINITY)) return MPSBNB_ERR_INVALID_ARG;
    if (q_token_stride < 0 || q_head_stride < 0) return MPSBNB_ERR_INVALID_ARG;
    if (seqs->batch == 0 || seqs->tokens == 0) return MPSBNB_OK;
    if (q == nullptr || out == nullptr) return MPSBNB_ERR_INVALID_ARG;
    const int group = heads / cache->kv_heads;
    // rows of a sequence and head are 32-bit numbers, with room for the tile behind the last (outputs of 2^31 rows: 256 GB and more)
    if (seqs->tokens * group > 0x7ffff000ll) return MPSBNB_ERR_TOO_LARGE;
    if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < mpsbnb_attention_4bit_workspace_bytes(cache, seqs, heads)) return MPSBNB_ERR_WORKSPACE;
    // rows are fetched in 16-byte pieces
    if (!aligned16(q) || ((q_token_stride | q_head_stride) & 7) != 0 || !aligned16(out)) return MPSBNB_ERR_UNSUPPORTED;
    Attn4Args a;
    a.kv = kv4_layer(cache, layer);
    a.sq = kv4_seqs(seqs, cache);
    a.q = q; a.q_ts = q_token_stride; a.q_hs = q_head_stride;
    a.out = out; a.lse = lse; a.ws = (float *)workspace;
    a.heads = heads; a.group = group; a.causal = causal != 0; a.window = window < (1 << 30) ? window : 1 << 30; a.quant_type = cache->quant_type;
    a.scale_log2 = scale * 1.4426950408889634f;
    static const float codes[2][16] = {MPSBNB_NF4_TABLE, MPSBNB_FP4_TABLE};
    for (int i = 0; i < 16; ++i) a.code[i] = codes[cache->quant_type][i] * attn4_code_scale(cache->quant_type);
    a.rows_lo = 0; a.rows_hi = 0x7fffffff;
    a.wide = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(workspace) + ad_tokens_ws(cache, seqs, group));
    a.wide_n = a.redo = 0;
    cudaStream_t st = (cudaStream_t)stream;
    const AdPlan plan = ad_plan(cache, seqs, group, window);
    if (plan.prompts != AD_TOKENS) {
        if (plan.mixed) a.rows_lo = ad_few_rows(cache->head_dim);
        rc = ad_prompt(a, cache, plan.prompts == AD_PROMPTS_SPLIT, st);
        if (rc != MPSBNB_ERR_UNSUPPORTED && (rc != MPSBNB_OK || !plan.mixed)) return rc;
        if (rc == MPSBNB_OK) a.rows_hi = a.rows_lo;                  // (else nothing has been launched: the kernel here takes all)
        a.rows_lo = 0;
    }
    return ad_run(a, cache, plan.nt, st);
}

extern "C" int mpsbnb_attention_4bit_kernels(const mpsbnb_kv4_cache *cache, const mpsbnb_kv4_seqs *seqs, int heads, int window) {
    int rc = kv4_check_cache(cache, 0);
    if (rc == MPSBNB_OK) rc = kv4_check_seqs(seqs, cache);
    if (rc != MPSBNB_OK) return rc;
    if (heads <= 0 || heads % cache->kv_heads != 0 || window < 0) return MPSBNB_ERR_INVALID_ARG;
    if (seqs->batch == 0 || seqs->tokens == 0) return 0;
    const AdPlan plan = ad_plan(cache, seqs, heads / cache->kv_heads, window);
    return (plan.mixed || plan.prompts == AD_TOKENS ? MPSBNB_ATTENTION_TOKENS : 0) | (plan.prompts != AD_TOKENS ? MPSBNB_ATTENTION_PROMPTS : 0) |
           (plan.prompts == AD_PROMPTS_SPLIT ? MPSBNB_ATTENTION_SHARED_OUT : 0);
}
