// Attention under a mask for many query rows, on the 5th-generation tensor
// cores: sliding windows with sinks, trees of drafted tokens.
//
// Work: items of (sequence, kv head, up to 256 query rows: whole tokens) x the
// 128-key tiles that any of its rows sees, a windowed item's sink tiles first.
// Items lie end to end on a line that is cut into equal runs, one per CTA (one
// CTA per SM), each item as long as it has tiles.
//
// A CTA runs two streams, A and B, each with its own rows of Q, two buffers for the
// scores of 64 keys (weights overwrite their scores, two 16-bit pieces each) and its own
// accumulator in TMEM.  With more than 128 rows each has half of them and takes both
// halves of every tile; with up to 128 both take the same rows, A the first half of
// each tile and B the second, and the accumulators, side by side in TMEM, are joined
// when the item ends.  The tensor core is two steps of scores ahead of a stream's
// softmax: PV_A(i), S_A(i + 2) | PV_B(i), S_B(i + 2) | ...  (With one buffer of 128
// keys a stream's softmax waited for its own PV and S: 5.0k cycles for a tile of both
// streams, in which the tensor core was busy for 2.6k.)
//
// Masks: a tile that some row does not see whole has its scores set to minus
// infinity in TMEM by two cuts (windowed) or by the node's ancestors (a tree),
// whose tiles are few; other tiles take no test.  An infinity or NaN among values
// that a row does not see must not meet its zero weight: a warp of its own looks
// through the masked tiles' values, puts zeros in their place and notes where they
// were, and a row that does see one has a NaN in that channel at the end.
//
// Bound: the tensor core and the softmax beside it.  A step of 64 keys of both streams is the scores, 2 x 128 x 64 x D, and
// twice that for the two pieces of the weights: 1536 cycles at D = 128 at the pipe's rate of 4096 products a cycle; beside
// them 128 x 64 exponentials a stream, 1024 cycles of the function unit.  What is longer than either is the chain score,
// weights, product of a stream.  Windows of 8064 keys for 4736 tokens: 372 us, 841 TFLOP/s (a weight's product counted once),
// 0.50 of cuBLAS.  8 prompts of 2000 in a window of 1024: 206 us, 0.24: an item's 128 tokens see 1024 keys each in 10 or 11
// tiles of 128, three or four of them masked and their values looked through, and items are short against their start and
// end.  32 trees of 64 on 8192: 171 us here and 10 in the join, alone; 811 MB of K and V at 4.7 TB/s, 0.72 of the copy rate,
// the tensor pipe active 49 % of the time.  One piece a weight was 338, 174 and 154 us.
//
// Tried: tiles prefetched into L2, 128 keys in one buffer, rolled loops over the MMAs, MMA code specialised by case: all slower.
//
// An item that a run's end cuts leaves a part (m, l, acc) per row and run, which
// the join adds in the order of the positions.
#pragma once

#include "paged_prefix.cuh"

namespace mq {
namespace paged {

constexpr int SPAN_THREADS = 384;   // warps: 0 items and K, 1 MMA of A, 2 Q and V (loads, and looks through V), 3 MMA of B, 4-7 softmax of A, 8-11 of B
constexpr int HK = 64;              // keys to a step of a stream
constexpr int SPAN_SEQS = 448;      // sequences of a call: their schedule is in shared memory
constexpr int SPAN_ITEMS = 4;       // ring of items between the first warp and the others

template <int D>
struct SpanSmem {
    static constexpr int TILE = (D / 64) * PATOM;
    static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE, BAR = 6 * TILE;
    static constexpr int ITEM = BAR + 512;                    // SpanSeg [SPAN_ITEMS]
    static constexpr int SUM = ITEM + SPAN_ITEMS * 64;        // fp32 [2 streams][128] row sums
    static constexpr int TOP = SUM + 2 * 128 * 4;             // fp32 [2 streams][128] their reference
    static constexpr int HIT = TOP + 2 * 128 * 4;             // u64 [2 streams][128][2]: channels in which a row met a value that is not finite
    static constexpr int ODD = HIT + 2 * 128 * 16;            // [2 stages][128 keys][D / 8]: a bit for each such value
    static constexpr int STAGE = ODD + 2 * 128 * (D / 8);     // [8 warps][32 rows][64 bytes] of the output
    static constexpr int SCHED = STAGE + 8 * 2048;
    static constexpr size_t bytes(int B) { return SCHED + (size_t)(4 * B + 2) * 4 + 1024; }
};

// the limit of a CTA, with the kernel's own sums of a warp
static_assert(SpanSmem<128>::bytes(SPAN_SEQS) + SPAN_THREADS / 32 * sizeof(unsigned long long) <= 227 * 1024,
              "the schedule of SPAN_SEQS sequences");

// An item that is cut: the worker with its first tile leaves this for the join.
struct alignas(16) SpanCut {
    int tok0, h, rows, runs;   // rows 0: none
};

struct alignas(16) SpanSeg {
    int slot, h, tok0, rows;      // tok0: the tile's first token; rows: of this item
    int seq0, pf, pl;             // the sequence's first token; positions of the tile's first and last token
    int st, wt, ng;               // sink tiles, first window tile, tiles in all
    int t0, n, runs;              // of this run (n 0: the run is over); runs that share the item
    bool two, start, whole;       // two: each stream has rows of its own
};
static_assert(sizeof(SpanSeg) <= 64, "an item of the ring");

// Tiles of a row tile whose tokens stand at pf .. pl: st of the sinks, then wt .. the one of pl.
__device__ __forceinline__ int span_tiles(const RowArgs& a, int pf, int pl, int& st, int& wt) {
    st = wt = 0;
    if (pl < 0) return 0;
    const int end = (pl >> 7) + 1;
    if (a.window) {
        wt = max(pf - a.window + 1, 0) >> 7;
        st = min(a.sinks > 0 ? ((a.sinks - 1) >> 7) + 1 : 0, wt);
    }
    return st + end - wt;
}

// 64 positions from `at` on that a row at position p sees; node: its place in the tree whose first token is seq0.
__device__ __forceinline__ unsigned long long span_sees(const RowArgs& a, int p, int at, int node, int seq0) {
    auto low = [](int k) { return k >= 64 ? ~0ull : k <= 0 ? 0ull : (1ull << k) - 1ull; };
    if (!a.parents) return low(p + 1 - at) & (~low(p + 1 - a.window - at) | low(a.sinks - at));
    const int base = p - node;
    unsigned long long bits = low(base - at);
    if (at + 64 <= base) return bits;
    while (node >= 0) {
        const int i = base + node - at;
        if (i >= 0 && i < 64 && base + node >= 0) bits |= 1ull << i;
        const int up = __ldg(a.parents + seq0 + node);
        if (up >= node || up < -1) note_status(a.status, MQ_ERR_INVALID_ARGUMENT);
        node = up >= node ? -1 : up;
    }
    return bits;
}

__device__ __forceinline__ void tma_load_heads(uint32_t dst, const CUtensorMap* map, int block, int head, int token, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(0), "r"(block), "r"(head), "r"(token), "r"(bar)
        : "memory");
}
// Operands in the 128-byte swizzle layout as sw128_kmajor_desc and sw128_mnmajor_desc have them: low word (address and
// leading offset, in units of 16 bytes) and the high word that is alike for both.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t leading) { return ((addr >> 4) & 0x3fffu) | leading << 16; }
constexpr uint32_t DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"((uint32_t)add), "n"(DESC_HI)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "mov.b64 b, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"((uint32_t)add), "n"(DESC_HI)
        : "memory");
}
// As mbar_try_wait, but answers at once (try_wait may hold the thread for some microseconds).
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Two fp32 values side by side.
__device__ __forceinline__ uint64_t two_of(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void halves(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <typename T, int D>
__global__ void __launch_bounds__(SPAN_THREADS, 1)
span_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
            const __grid_constant__ CUtensorMap tmV, const RowArgs a, SpanCut* __restrict__ cuts) {
    using L = SpanSmem<D>;
    constexpr int TILE = L::TILE, LD = D + 4, NT = SPAN_THREADS;
    extern __shared__ uint8_t pfx_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pfx_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR);
    uint64_t* q_full = bars;          // [2] streams
    uint64_t* k_full = bars + 2;      // [2] stages
    uint64_t* k_empty = bars + 4;
    uint64_t* v_full = bars + 6;
    uint64_t* v_empty = bars + 8;
    uint64_t* v_ready = bars + 10;    // [2] stages: looked through
    uint64_t* s_full = bars + 12;     // [2 streams][2 buffers] scores are there
    uint64_t* p_full = bars + 16;     // [2][2] weights are stored, O is rescaled
    uint64_t* o_full = bars + 20;     // [2] the PV of an item's last step but one is done, and that of the last
    uint64_t* q_empty = bars + 22;    // [2]
    uint64_t* drain = bars + 24;
    uint64_t* pair = bars + 25;       // [4] the warps of A and B on the same rows
    uint64_t* item_full = bars + 29;  // [SPAN_ITEMS]
    uint64_t* item_empty = item_full + SPAN_ITEMS;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(item_empty + SPAN_ITEMS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
    volatile int* holes = abort_flag + 1;      // a page out of range has been met
    volatile int* odd_tile = abort_flag + 2;   // [2] stages: the tile holds values that are not finite
    __shared__ unsigned long long scratch[NT / 32];
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 2);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 2);
            mbar_init(&v_ready[i], 1);
            mbar_init(&s_full[2 * i], 1);
            mbar_init(&s_full[2 * i + 1], 1);
            mbar_init(&p_full[2 * i], 4);
            mbar_init(&p_full[2 * i + 1], 4);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(drain, 2);
        for (int i = 0; i < 4; ++i) mbar_init(&pair[i], 2);
        for (int i = 0; i < SPAN_ITEMS; ++i) {
            mbar_init(&item_full[i], 1);
            mbar_init(&item_empty[i], NT / 32 - 1);
        }
        *abort_flag = 0;
        *holes = 0;
        fence_mbar_init();
        prefetch_tmap(&tmQ);
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    if (warp == 1) {
        tmem_alloc(tmem_holder, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    pdl_wait();
    pdl_trigger();

    // ---- the line: off[b] units before sequence b, for one kv head ----
    uint32_t* off = reinterpret_cast<uint32_t*>(smem + L::SCHED);   // [B + 1]
    int* first = reinterpret_cast<int*>(off + a.B + 1);             // [B + 1] query tokens before
    int* lens = first + a.B + 1;                                    // [B], 0 where nothing is read
    int* slots = lens + a.B;                                        // [B]
    const int grp = a.grp, page = a.pool.page, tps = PROWS / 2 / grp, tpt = 2 * tps;   // tokens to a stream and to a row tile
    constexpr uint32_t LATER = 0xffffffffu;   // a sequence of many row tiles: their costs are summed by a warp
    bool bad = false, later = false;
    for (int b = threadIdx.x; b <= a.B; b += NT) {
        const int q0 = q_start(a, b);
        first[b] = q0;
        if (b == a.B) {
            bad |= q0 != a.total_q;
            break;
        }
        const int slot = __ldg(a.slots + b), ql = q_start(a, b + 1) - q0;
        bad |= ql < 0 || (b == 0 && q0 != 0);
        int len = 0, code = 0;
        if (slot < 0 || slot >= a.num_slots) {
            code = MQ_ERR_BAD_SLOT;
        } else {
            len = __ldg(a.lengths + slot);
            if (len < 0 || pages_for(len, a.pool.shift) > a.cols) code = MQ_ERR_BAD_POSITION;
            else if (a.parents && ql > MAX_TREE) code = MQ_ERR_INVALID_ARGUMENT;
        }
        if (code) {
            len = 0;
            if (blockIdx.x == 0 && ql >= 0) note_status(a.status, code);
        }
        lens[b] = len;
        slots[b] = slot;
        uint32_t cost = 0;
        if (len && ql > 0) {
            if (ql > 4 * tpt) {
                cost = LATER;
                later = true;
            } else {
                int st, wt;
                for (int i = 0; i < ql; i += tpt) {
                    const int n = span_tiles(a, len - ql + i, len - ql + min(i + tpt, ql) - 1, st, wt);
                    cost += n ? n + ITEM_UNITS : 0;
                }
            }
        }
        off[b] = cost;
    }
    bool in_order = !__syncthreads_or(bad);
    if (__syncthreads_or(later && in_order)) {
        for (int b = warp; b < a.B; b += NT / 32) {
            if (off[b] != LATER) continue;
            const int ql = first[b + 1] - first[b], p0 = lens[b] - ql;
            unsigned long long cost = 0;
            for (int i0 = lane; (long long)i0 * tpt < ql; i0 += 32) {
                const int i = i0 * tpt;
                int st, wt;
                const int n = span_tiles(a, p0 + i, p0 + min(i + tpt, ql) - 1, st, wt);
                cost += n ? n + ITEM_UNITS : 0;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) cost += __shfl_xor_sync(0xffffffffu, cost, o);
            __syncwarp();
            if (lane == 0) off[b] = (uint32_t)(cost < 0x7fffffffull ? cost : 0x7fffffffull);   // (a sum that long is refused below)
        }
        __syncthreads();
    }
    {
        unsigned long long carry = 0;
        for (int b0 = 0; in_order && b0 < a.B; b0 += NT) {
            const int b = b0 + threadIdx.x;
            const unsigned long long cost = b < a.B ? off[b] : 0;
            unsigned long long x = cost;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (lane == 31) scratch[warp] = x;
            __syncthreads();
            unsigned long long before = carry;
            for (int w = 0; w < NT / 32; ++w) {
                const unsigned long long v = scratch[w];
                if (w < warp) before += v;
                carry += v;
            }
            if (b < a.B) off[b] = (uint32_t)(before + x - cost);
            __syncthreads();
        }
        if (carry * (unsigned)a.hkv >= 0x7fffffffull) in_order = false;
        if (threadIdx.x == 0) off[a.B] = (uint32_t)carry;
    }
    __syncthreads();
    if (!in_order && blockIdx.x == 0 && threadIdx.x == 0) note_status(a.status, MQ_ERR_INVALID_ARGUMENT);
    const uint32_t work = in_order ? off[a.B] * a.hkv : 0, quota = quota_of(work, gridDim.x);
    const uint32_t x0 = min(blockIdx.x * quota, work), xe = min(x0 + quota, work);

    // The run's items in order, by the first warp: the first one is looked up, the others follow it.
    int it_b = 0, it_h = 0, it_i = 0, it_ql = 0, it_p0 = 0;   // sequence, head, the row tile's first token; of the sequence
    uint32_t x = x0;
    SpanSeg cur;
    auto open = [&](int b) {
        it_b = b;
        cur.slot = slots[b];
        cur.seq0 = first[b];
        it_ql = first[b + 1] - cur.seq0;
        it_p0 = lens[b] - it_ql;
    };
    auto locate = [&]() -> int {   // units of the item before x
        const uint32_t xh = x / (uint32_t)a.hkv;
        int lo = 0, hi = a.B;   // the last sequence that starts at or before, of those with work
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (off[mid] <= xh) lo = mid;
            else hi = mid;
        }
        open(lo);
        const uint32_t one = off[lo + 1] - off[lo];
        uint32_t rel = x - off[lo] * a.hkv;
        it_h = (int)(rel / one);
        rel -= it_h * one;
        for (int i0 = 0;; i0 += 32) {   // the row tile, 32 at a time
            const int i = (i0 + lane) * tpt;
            int st, wt, n = 0;
            if (i < it_ql) n = span_tiles(a, it_p0 + i, it_p0 + min(i + tpt, it_ql) - 1, st, wt);
            const uint32_t cost = n ? n + ITEM_UNITS : 0;
            uint32_t sum = cost;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += y;
            }
            const unsigned found = __ballot_sync(0xffffffffu, rel < sum);
            if (!found && (i0 + 32) * tpt < it_ql) {
                rel -= __shfl_sync(0xffffffffu, sum, 31);
                continue;
            }
            const int at = found ? __ffs((int)found) - 1 : 0;   // (always found: x is within the sequence)
            rel -= __shfl_sync(0xffffffffu, sum - cost, at);
            it_i = (i0 + at) * tpt;
            return (int)rel;
        }
    };
    auto follow = [&]() {   // to the next row tile, head or sequence; x is on the line's work
        it_i += tpt;
        if (it_i < it_ql) return;
        it_i = 0;
        if (++it_h < a.hkv) return;
        it_h = 0;
        int b = it_b + 1;
        while (off[b + 1] == off[b]) ++b;
        open(b);
    };
    // The next item with tiles in this run, into cur; n = 0 at the run's end.
    bool placed = false;
    auto next_item = [&]() {
        cur.n = 0;
        while (x < xe && cur.n <= 0) {
            int pos = 0;
            if (!placed) pos = locate();
            else follow();
            placed = true;
            const int last = min(it_i + tpt, it_ql) - 1;
            cur.h = it_h;
            cur.tok0 = cur.seq0 + it_i;
            cur.rows = (last - it_i + 1) * grp;
            cur.pf = it_p0 + it_i;
            cur.pl = it_p0 + last;
            cur.ng = span_tiles(a, cur.pf, cur.pl, cur.st, cur.wt);
            if (!cur.ng) continue;   // (before the first position)
            const int left = (int)min((uint32_t)(cur.ng + ITEM_UNITS - pos), xe - x);
            cur.t0 = max(pos - ITEM_UNITS, 0);
            cur.n = max(pos + left - ITEM_UNITS, 0) - cur.t0;
            cur.two = cur.rows > tps * grp;
            cur.start = cur.t0 == 0;
            cur.whole = cur.n == cur.ng;
            cur.runs = 1;
            if (!cur.whole) {
                const uint32_t ps = x - pos + ITEM_UNITS;   // the item's first tile on the line
                cur.runs = (int)((ps + cur.ng - 1) / quota - ps / quota) + 1;
            }
            x += left;
        }
    };
    auto tile_at = [&](const SpanSeg& e, int j) {   // first position of the run's j-th tile
        const int t = e.t0 + j;
        return (t < e.st ? t : e.wt + t - e.st) * PK;
    };
    // Every row sees all of the n keys at `at`.
    auto all_seen = [&](const SpanSeg& e, int at, int n) {
        if (a.parents) return at + n <= e.seq0 - e.tok0 + e.pf;
        return at + n - 1 <= e.pf && (at > e.pl - a.window || at + n <= a.sinks);
    };
    // Some row sees a position of the page at `at`: other pages' entries in the table are not looked at.
    auto in_sight = [&](const SpanSeg& e, int at) {
        return at <= e.pl && (a.parents || at < a.sinks || at + page > e.pf - a.window + 1);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (mbar_try_wait(bar, parity)) return true;
        const long long t0 = clock64();
        while (!mbar_try_wait(bar, parity)) {
            if (*abort_flag || clock64() - t0 > WAIT_CYCLES) return false;
        }
        return true;
    };
    auto give_up = [&]() {
        *abort_flag = 1;
        note_status(a.status, MQ_ERR_PIPE_TIMEOUT);
    };
    // The other warps' items, in the order in which the first one leaves them; false at the end of the run.
    SpanSeg* items = reinterpret_cast<SpanSeg*>(smem + L::ITEM);
    auto item_at = [&](int i) -> SpanSeg& { return *reinterpret_cast<SpanSeg*>(reinterpret_cast<uint8_t*>(items) + (i % SPAN_ITEMS) * 64); };
    int taken = 0;
    auto take = [&](SpanSeg& e, bool& ok) {
        ok = ok && __all_sync(0xffffffffu, wait(&item_full[taken % SPAN_ITEMS], (taken / SPAN_ITEMS) & 1));
        if (!ok) return false;
        e = item_at(taken);
        return e.n > 0;
    };
    auto done_with = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[taken % SPAN_ITEMS]);
        ++taken;
    };

    // copies in flight land before the CTA may end, whatever became of their readers
    auto land = [&](uint64_t* bar, uint32_t parity) {
        const long long t0 = clock64();
        while (!mbar_try_wait(bar, parity) && clock64() - t0 < WAIT_CYCLES) {
        }
    };
    // Page `c` of a tile for lane c: what no row sees is read as zeros, from outside the map.
    const int chunks = PK / page;
    auto look = [&](const SpanSeg& e, int j) {
        const int at = tile_at(e, j) + lane * page;
        if (lane >= chunks || !in_sight(e, at)) return a.pool.pages;
        return __ldg(a.table + e.slot * a.table_row + (at >> a.pool.shift));
    };
    auto load_tile = [&](const SpanSeg& e, int j, int pid, const CUtensorMap* map, uint8_t* to, uint64_t* full) {
        if (pid < 0 || pid >= a.pool.pages) {
            if (lane < chunks && in_sight(e, tile_at(e, j) + lane * page)) {
                note_status(a.status, MQ_ERR_BAD_PAGE);
                *holes = 1;   // before the tile's scores are there
            }
            pid = a.pool.pages;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(full, TILE);
        __syncwarp();
        if (lane < chunks) {
#pragma unroll
            for (int i = 0; i < D / 64; ++i)
                tma_load_page(smem_u32(to + i * PATOM + lane * page * 128), map, 0, i, e.h, pid, smem_u32(full));
        }
    };

    if (warp == 0) {
        // ---- the items, and K ----
        int c = 0;   // tiles so far
        bool ok = true, cut = false;
        while (ok) {
            next_item();
            if (taken >= SPAN_ITEMS)
                ok = __all_sync(0xffffffffu, wait(&item_empty[taken % SPAN_ITEMS], (taken / SPAN_ITEMS - 1) & 1));
            if (!ok) break;
            if (lane == 0) {
                item_at(taken) = cur;
                mbar_arrive(&item_full[taken % SPAN_ITEMS]);
            }
            ++taken;
            if (cur.n <= 0) break;
            if (cur.start && !cur.whole) {   // (the run's last item)
                if (lane == 0) *reinterpret_cast<int4*>(cuts + blockIdx.x) = make_int4(cur.tok0, cur.h, cur.rows, cur.runs);
                cut = true;
            }
            int next = look(cur, 0);
            for (int j = 0; j < cur.n; ++j, ++c) {
                const int pid = next, st = c & 1;
                if (j + 1 < cur.n) next = look(cur, j + 1);
                if (c >= 2) ok = __all_sync(0xffffffffu, wait(&k_empty[st], ((c >> 1) - 1) & 1));
                if (!ok) break;
                load_tile(cur, j, pid, &tmK, smem + L::K + st * TILE, &k_full[st]);
            }
        }
        if (!cut && lane == 0) *reinterpret_cast<int4*>(cuts + blockIdx.x) = make_int4(0, 0, 0, 0);
        if (!ok && lane == 0) give_up();
        for (int k = max(0, c - 2); k < c; ++k) land(&k_full[k & 1], (k >> 1) & 1);
    } else if (warp == 2) {
        // ---- Q and V: loads, and what is looked through when it has landed.  Whatever is waited for, tiles of V that land
        // meanwhile are passed on ----
        int c = 0, seen = 0, nq = 0;   // tiles asked for, tiles passed on, items
        uint32_t masked = 0;           // bit st: the tile in stage st is not seen whole by every row
        bool ok = true;
        auto pass_on = [&]() {
            const int st = seen & 1;
            if (masked >> st & 1u) {
                constexpr uint32_t M = Elem<T>::EXP_MASK * 0x10001u, U = (Elem<T>::EXP_MASK & -Elem<T>::EXP_MASK) * 0x10001u;
                uint8_t* vt = smem + L::V + st * TILE;
                uint32_t any = 0;
#pragma unroll 8
                for (int i = lane; i < TILE / 16; i += 32) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vt + i * 16);
                    // an exponent of all ones and one more carries out of its field
                    any |= ((w.x & M) + U) | ((w.y & M) + U) | ((w.z & M) + U) | ((w.w & M) + U);
                }
                const bool odd = __any_sync(0xffffffffu, any & 0x80008000u);
                if (odd) {
                    uint8_t* bits = smem + L::ODD + st * 128 * (D / 8);
                    for (int i = lane; i < TILE / 16; i += 32) {
                        // 16-byte piece i: block of 64 channels, key, piece of it (swizzled by the key)
                        const int key = i >> 3 & 127, ch = (i >> 10) * 8 + ((i & 7) ^ (key & 7));
                        uint4 w = *reinterpret_cast<const uint4*>(vt + i * 16);
                        uint32_t* v = reinterpret_cast<uint32_t*>(&w);
                        uint32_t mark = 0;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t f = (v[k] & M) + U;
                            if (f & 0x8000u) mark |= 1u << (2 * k), v[k] &= 0xffff0000u;
                            if (f & 0x80000000u) mark |= 2u << (2 * k), v[k] &= 0xffffu;
                        }
                        bits[key * (D / 8) + ch] = (uint8_t)mark;
                        if (mark) *reinterpret_cast<uint4*>(vt + i * 16) = w;
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                if (lane == 0) odd_tile[st] = odd;
                __syncwarp();
            }
            if (lane == 0) mbar_arrive(&v_ready[st]);
            ++seen;
        };
        auto pump = [&](uint64_t* bar, uint32_t parity) {   // waits for bar
            const long long t0 = clock64();
            while (ok && !__all_sync(0xffffffffu, mbar_test_wait(bar, parity & 1))) {
                if (seen < c && __all_sync(0xffffffffu, mbar_test_wait(&v_full[seen & 1], (seen >> 1) & 1))) pass_on();
                if (__any_sync(0xffffffffu, *abort_flag || clock64() - t0 > WAIT_CYCLES)) ok = false;
            }
            return ok;
        };
        for (SpanSeg e; pump(&item_full[taken % SPAN_ITEMS], taken / SPAN_ITEMS) && take(e, ok); ++nq) {
            done_with();
            for (int q = 0; q < 2; ++q) {
                if (nq && !pump(&q_empty[q], nq - 1)) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&q_full[q], (D / 64) * tps * grp * 128);
#pragma unroll
                    for (int i = 0; i < D / 64; ++i)
                        tma_load_heads(smem_u32(smem + L::Q + q * TILE + i * PATOM), &tmQ, i, e.h * grp,
                                       e.tok0 + (e.two ? q * tps : 0), smem_u32(&q_full[q]));
                }
            }
            if (!ok) break;
            int next = look(e, 0);
            for (int j = 0; j < e.n; ++j) {
                const int pid = next, st = c & 1;
                if (j + 1 < e.n) next = look(e, j + 1);
                if (c >= 2 && !pump(&v_empty[st], (c >> 1) - 1)) break;
                masked = (masked & ~(1u << st)) | (uint32_t)!all_seen(e, tile_at(e, j), PK) << st;
                load_tile(e, j, pid, &tmV, smem + L::V + st * TILE, &v_full[st]);
                ++c;
            }
        }
        while (ok && seen < c) {
            ok = __all_sync(0xffffffffu, wait(&v_full[seen & 1], (seen >> 1) & 1));
            if (ok) pass_on();
        }
        if (!ok) {
            if (lane == 0) give_up();
            for (int k = max(0, c - 2); k < c; ++k) land(&v_full[k & 1], (k >> 1) & 1);
            // (otherwise the scores of every Q tile have been waited for)
            for (int q = 0; q < 2; ++q)
                if (nq) land(&q_full[q], (nq - 1) & 1);
            land(&q_full[0], nq & 1);   // A's of an item whose B could not be asked for (if there is none, this runs out)
        }
    } else if (warp == 1 || warp == 3) {
        // ---- MMA of a stream: the whole warp walks, one elected lane issues.  All 512 columns of TMEM are this CTA's, so
        // their addresses start at 0.  The tensor core takes an MMA when the one before is nearly done (12 MMAs of 620
        // cycles take 620 to issue to an idle pipe), so what an issuing warp does between two is lost to the pipe unless
        // another warp issues meanwhile: a warp for each stream ----
        const int q = warp >> 1;
        constexpr uint32_t id_o = pfx_idesc<T>(D, true);
        // a negative scale: the scores of -Q
        const uint32_t id_s = pfx_idesc<T>(HK, false) | (a.scale_log2 < 0.f ? 1u << 13 : 0u);
        const uint32_t base = (smem_u32(pfx_raw) + 1023u) & ~1023u;
        int c0 = 0;          // tiles of the items before
        uint32_t g = 0;      // steps (64 keys) of the items before
        uint32_t nq = 0;     // items
        bool ok = true;
        const uint32_t q_lo = desc_lo(base + L::Q, 1) + q * (TILE >> 4);
        const uint32_t k_lo = desc_lo(base + L::K, 1), v_lo = desc_lo(base + L::V, PATOM >> 4);
        for (SpanSeg e; take(e, ok); done_with()) {
            const bool two = uniform(e.two);
            const int n = uniform(e.n), steps = two ? 2 * n : n;
            // steps -2 and -1: scores of steps 0 and 1; step i: PV of step i, then scores of step i + 2, whose buffer
            // the weights of step i were in.  What a step needs is waited for by four lanes at once.
            for (int i = -2; ok && i < steps; ++i) {
                const bool pv = i >= 0, sc = i + 2 < steps;
                const int vc = c0 + (two ? i >> 1 : i), kc = c0 + (two ? (i + 2) >> 1 : i + 2);
                if (!pv && !sc) continue;   // (an item of one step)
                uint64_t* bar = nullptr;
                uint32_t parity = 0;
                if (lane == 0 && sc) bar = &k_full[kc & 1], parity = kc >> 1;
                if (lane == 1 && pv) bar = &v_ready[vc & 1], parity = vc >> 1;
                if (lane == 2 && pv) bar = &p_full[2 * q + ((g + i) & 1)], parity = (g + i) >> 1;
                if (lane == 3 && i == -2) bar = &q_full[q], parity = nq;
                ok = __all_sync(0xffffffffu, !bar || wait(bar, parity & 1));
                if (!ok) break;
                tc_fence_after();
                // a stream takes both halves of a tile, or one
                const int half = two ? i & 1 : q;
                const bool used = !two || (i & 1);
                const uint32_t buffer = q * 128 + ((g + i) & 1) * HK, o = 256 + q * 128;
                const uint32_t vl = v_lo + (vc & 1) * (TILE >> 4) + half * (HK * 128 >> 4);
                const uint32_t kl = k_lo + (kc & 1) * (TILE >> 4) + half * (HK * 128 >> 4);
                if (elect_one()) {
                    if (pv) {
#pragma unroll
                        for (int k = 0; k < HK / 16; ++k) {   // 16 keys: 8 columns of weights, 8 of their second pieces
                            mma_ts(o, buffer + 8 * k, vl + k * (2048 >> 4), id_o, k || i);
                            mma_ts(o, buffer + HK / 2 + 8 * k, vl + k * (2048 >> 4), id_o, true);
                        }
                        if (i + 2 >= steps) tc_commit(&o_full[q]);
                        if (used) tc_commit(&v_empty[vc & 1]);
                    }
                    if (sc) {
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const uint32_t x = ((k >> 2) * PATOM + (k & 3) * 32) >> 4;
                            mma_ss(buffer, q_lo + x, kl + x, id_s, k != 0);
                        }
                        tc_commit(&s_full[2 * q + ((g + i) & 1)]);
                        if (used) tc_commit(&k_empty[kc & 1]);
                        if (i + 3 == steps) tc_commit(&q_empty[q]);
                    }
                }
                __syncwarp();
            }
            c0 += n;
            g += steps;
            ++nq;
        }
        if (!ok && lane == 0) give_up();
        if (elect_one()) tc_commit(drain);   // MMAs in flight end before TMEM goes
        __syncwarp();
        const long long t0 = clock64();
        while (!mbar_try_wait(drain, 0) && clock64() - t0 < WAIT_CYCLES) {
        }
    } else {
        // ---- softmax of stream q: a thread to a row ----
        const int q = (warp - 4) >> 2, quad = warp & 3;   // quad: the TMEM lanes this warp may touch
        const int r = quad * 32 + lane;
        // a scale of zero: a masked score of minus infinity stays one
        const float scale = fmaxf(fabsf(a.scale_log2), 1e-30f);
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const uint32_t sa = tmem + lane_off + q * 128, oa = tmem + lane_off + 256;   // O of A, that of B 128 columns on
        float* sums = reinterpret_cast<float*>(smem + L::SUM);   // [stream][128]
        float* tops = reinterpret_cast<float*>(smem + L::TOP);
        uint8_t* stage = smem + L::STAGE + (warp - 4) * 2048;
        ulonglong2* hits = reinterpret_cast<ulonglong2*>(smem + L::HIT);
        // fp16 ends 24 octaves below 1 and 16 above it: weights stand 5 octaves higher there and may grow to 2^15.5, so that what
        // is lost of one is at most 2^-30 of the row's largest, and 2^17 of them are 2^-13 of it.  8 prompts of 2000, as the
        // sums are rescaled more often the less room is left: 5 octaves 202 us, 6 211, 10 239.
        constexpr bool HALF = Elem<T>::MAX < 1e5f;
        constexpr float GROW = HALF ? 15.5f : 14.f, BELOW = HALF ? 5.f : 0.f;
        uint32_t g = 0, no = 0;  // steps (64 keys) so far, alike for both streams; o_full so far
        int nv = 0, np = 0;      // tiles of the items before, meetings
        bool ok = true;
        auto got = [&](uint64_t* bar, uint32_t parity) {
            if (ok) ok = __all_sync(0xffffffffu, wait(bar, parity & 1));
            return ok;
        };
        auto meet = [&]() {   // with the other stream's warp on the same rows
            __syncwarp();
            if (lane == 0) mbar_arrive(&pair[quad]);
            got(&pair[quad], np++);
        };
        const int tok_r = r / grp, head_r = r - tok_r * grp;   // of this row in its stream
        for (SpanSeg e; take(e, ok); done_with()) {
            const int steps = e.two ? 2 * e.n : e.n;
            const int tok = (e.two ? q * tps : 0) + tok_r;       // the row's token in the item
            const bool there = tok_r < tps && tok * grp < e.rows;
            const int pos = min(e.pf + tok, e.pl), node = e.tok0 - e.seq0 + pos - e.pf;
            unsigned long long hit[2] = {0, 0};
            float m = -INFINITY, l = 0.f;
#pragma unroll 1
            for (int i = 0; i < steps; ++i, ++g) {
                const int jt = e.two ? i >> 1 : i, tile = tile_at(e, jt), at = tile + (e.two ? i & 1 : q) * HK;
                const bool looked = !all_seen(e, tile, PK);   // through the tile's values
                unsigned long long live = ~0ull;              // keys that the row sees
                if (looked && !all_seen(e, at, HK)) live = span_sees(a, pos, at, node, e.seq0);
                const uint32_t sb = sa + (g & 1) * HK;
                if (!got(&s_full[2 * q + (g & 1)], g >> 1)) break;
                tc_fence_after();
                const int hole = *holes;
                float sv[HK];
                tmem_ld64(sb, sv);
                if (hole) {   // pages out of range: their keys are left out
                    const int* row = a.table + e.slot * a.table_row;
                    for (int k = 0; k < HK; k += min(page, HK)) {
                        const int p = (at + k) & -page;
                        const int pid = in_sight(e, p) ? __ldg(row + (p >> a.pool.shift)) : 0;
                        if (pid < 0 || pid >= a.pool.pages) live &= ~((page >= HK ? ~0ull : (1ull << page) - 1ull) << k);
                    }
                }
                if (looked || hole) {
                    const uint32_t lo = (uint32_t)live, hi = (uint32_t)(live >> 32);
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        sv[k] = lo >> k & 1u ? sv[k] : -INFINITY;
                        sv[32 + k] = hi >> k & 1u ? sv[32 + k] : -INFINITY;
                    }
                }
                float mx[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) mx[k] = fmaxf(sv[2 * k], sv[2 * k + 1]);
#pragma unroll
                for (int k = 8; k < HK; k += 2) mx[(k >> 1) & 3] = max3(mx[(k >> 1) & 3], sv[k], sv[k + 1]);
                const float tmax = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * scale;
                // a row's reference is its maximum (fp16: some octaves below it) and moves only when a maximum is many octaves above it:
                // weights stay below 2^GROW, and one of the first keys, among few, is often some octaves below the row's maximum
                float corr = 1.f;
                if (tmax > m + GROW) {
                    const float to = tmax - BELOW;
                    corr = m == -INFINITY ? 1.f : ex2(m - to);   // (nothing is summed before the first key that the row sees)
                    m = to;
                }
                l *= corr;
                if (i && __any_sync(0xffffffffu, corr != 1.f)) {
                    // O is at rest once the PV before is done: the scores after these came after it, or it was the last but one
                    if (i + 1 < steps ? !got(&s_full[2 * q + ((g + 1) & 1)], (g + 1) >> 1) : !got(&o_full[q], no)) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        float v[32];
                        tmem_ld32(oa + q * 128 + c, v);
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[k] *= corr;
                        tmem_st16_nowait(oa + q * 128 + c, reinterpret_cast<const uint32_t*>(v));
                        tmem_st16_nowait(oa + q * 128 + c + 16, reinterpret_cast<const uint32_t*>(v + 16));
                    }
                }
                const uint64_t scale2 = two_of(scale, scale), u2 = m == -INFINITY ? 0ull : two_of(-m, -m);
                const uint64_t minus1 = two_of(-1.f, -1.f);
                uint64_t sum0 = 0ull, sum1 = 0ull;
#pragma unroll
                for (int c = 0; c < HK; c += 32) {
                    // 32 weights in 16 columns and what they are short of in 16 more, over the scores: with one piece the
                    // result would be as far off as its own rounding
                    uint32_t pk[16], rest[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float p0, p1;
                        halves(fma2(two_of(sv[c + 2 * k], sv[c + 2 * k + 1]), scale2, u2), p0, p1);
                        p0 = ex2(p0);
                        p1 = ex2(p1);
                        const uint64_t both = two_of(p0, p1);
                        (k & 1 ? sum1 : sum0) = add2(k & 1 ? sum1 : sum0, both);
                        pk[k] = Elem<T>::pack(p0, p1);
                        const float2 b = Elem<T>::up2(pk[k]);
                        halves(fma2(two_of(b.x, b.y), minus1, both), p0, p1);
                        rest[k] = Elem<T>::pack(p0, p1);
                    }
                    tmem_st16_nowait(sb + (c >> 1), pk);
                    tmem_st16_nowait(sb + HK / 2 + (c >> 1), rest);
                }
                float s0, s1;
                halves(add2(sum0, sum1), s0, s1);
                l += s0 + s1;
                if (looked) {
                    // the tile's values are looked through, and stay until this stream's weights are used
                    const int c = nv + jt, st = c & 1;
                    if (got(&v_ready[st], c >> 1) && odd_tile[st]) {
                        const uint8_t* bits = smem + L::ODD + (st * 128 + at - tile) * (D / 8);
#pragma unroll 1
                        for (int k = 0; k < HK; ++k) {
                            if (!(live >> k & 1ull)) continue;
                            hit[0] |= *reinterpret_cast<const unsigned long long*>(bits + k * (D / 8));
                            if (D == 128) hit[1] |= *reinterpret_cast<const unsigned long long*>(bits + k * (D / 8) + 8 * (D / 128));
                        }
                    }
                }
                if (i && i + 1 == steps && !got(&o_full[q], no++)) break;   // (in its turn: a phase passed over cannot be told)
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[2 * q + (g & 1)]);
            }
            nv += e.n;
            // ---- the item's rows: what A and B have of them, when they share them ----
            got(&o_full[q], no++);
            tc_fence_after();
            float e0 = 1.f, e1 = 1.f;   // weights of A's and B's accumulators
            if (!e.two) {
                sums[q * 128 + r] = l;
                tops[q * 128 + r] = m;
                hits[q * 128 + r] = make_ulonglong2(hit[0], hit[1]);
                meet();   // (and the other stream's accumulator is complete, too)
                tc_fence_after();
                const float ma = tops[r], mb = tops[128 + r];
                m = fmaxf(ma, mb);
                const float u = m == -INFINITY ? 0.f : m;
                e0 = ex2(ma - u);
                e1 = ex2(mb - u);
                l = sums[r] * e0 + sums[128 + r] * e1;
                const ulonglong2 h0 = hits[r], h1 = hits[128 + r];
                hit[0] = h0.x | h1.x;
                hit[1] = h0.y | h1.y;
            }
            const float inv = l != 0.f ? 1.f / l : 0.f;   // a row that sees nothing is zero (NaN stays NaN)
            // this thread's columns: the row's, or with two streams on it half of them
            const int c_lo = e.two ? 0 : q * (D / 2), c_hi = e.two ? D : c_lo + D / 2;
            const uint32_t own = oa + (e.two ? q * 128 : 0);
            float* part = there ? a.ws.pfx_slots + ((2ll * blockIdx.x + e.start) * PROWS + tok * grp + head_r) * LD : nullptr;
            uint16_t* out = there ? a.out + ((long long)(e.tok0 + tok) * a.hq + e.h * grp + head_r) * D : nullptr;
            if (__any_sync(0xffffffffu, (hit[0] | hit[1]) != 0)) {   // channels in which a row met a value that is not finite
#pragma unroll 1
                for (int c = c_lo; ok && c < c_hi; c += 16) {
                    float v[16];
                    tmem_ld16(own + c, v);
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (hit[c >> 6] >> ((c & 63) + k) & 1ull) v[k] = NAN;
                    tmem_st16(own + c, v);
                }
            }
            uint16_t* rows[4];   // where this lane's piece of row 8 k + lane / 4 of the warp goes
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                rows[k] = from_lane(out, 8 * k + (lane >> 2));
                if (rows[k]) rows[k] += (lane & 3) * 8;
            }
            if (!e.whole && ok && there && (e.two || q == 0)) *reinterpret_cast<float4*>(part) = make_float4(m, l, 0.f, 0.f);
#pragma unroll 1
            for (int c = c_lo; ok && c < c_hi; c += 32) {
                float v[32];
                tmem_ld32(own + c, v);
                if (!e.two) {
                    float w[32];
                    tmem_ld32(oa + 128 + c, w);
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = v[k] * e0 + w[k] * e1;
                }
                if (!e.whole) {
                    if (there) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            *reinterpret_cast<float4*>(part + 4 + c + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                    }
                    continue;
                }
                // through shared memory (pieces of 16 bytes, swizzled), so that a store touches 64 bytes of each of eight
                // rows and not 16 of 32
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<uint4*>(stage + lane * 64 + ((k ^ (lane >> 1 & 3)) << 4)) =
                        make_uint4(Elem<T>::pack(v[8 * k] * inv, v[8 * k + 1] * inv), Elem<T>::pack(v[8 * k + 2] * inv, v[8 * k + 3] * inv),
                                   Elem<T>::pack(v[8 * k + 4] * inv, v[8 * k + 5] * inv), Elem<T>::pack(v[8 * k + 6] * inv, v[8 * k + 7] * inv));
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int row = 8 * k + (lane >> 2);
                    const uint4 w = *reinterpret_cast<const uint4*>(stage + row * 64 + (((lane & 3) ^ (row >> 1 & 3)) << 4));
                    if (rows[k]) *reinterpret_cast<uint4*>(rows[k] + c) = w;
                }
                __syncwarp();
            }
            tc_fence_before();
            if (!e.two) meet();   // both accumulators are read
        }
        if (!ok && lane == 0) give_up();
    }
    // rows that see nothing: sequences and row tiles without items (the whole call, when it is refused)
    {
        const int warps = gridDim.x * (NT / 32), wid = blockIdx.x * (NT / 32) + warp;
        auto clear = [&](int t0, int t1) {
            const long long words = (long long)(t1 - t0) * a.hq * (D / 8);
            uint4* to = reinterpret_cast<uint4*>(a.out) + (long long)t0 * a.hq * (D / 8);
            for (long long i = lane; i < words; i += 32) to[i] = make_uint4(0, 0, 0, 0);
        };
        if (!in_order) {
            for (int t = wid; t < a.total_q; t += warps) clear(t, t + 1);
        } else {
            for (int b = wid; b < a.B; b += warps) {
                const int t0 = first[b], ql = first[b + 1] - t0;
                int none = ql;   // tokens of row tiles that stand before the first position
                if (lens[b]) none = lens[b] >= ql ? 0 : min(ql, (ql - lens[b]) / tpt * tpt);
                if (none > 0) clear(t0, t0 + none);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// The join of the items that were cut: acc = sum acc_i 2^(m_i - M) over sum l_i 2^(m_i - M).  A warp to a row, blockIdx.y:
// eight rows of the cut.  (Four rows to a warp, one after the other, were four times the latency: 17 us for 148 cuts of 256.)
template <typename T, int D>
__global__ void __launch_bounds__(256) span_join_kernel(const RowArgs a, const SpanCut* __restrict__ cuts) {
    constexpr int LD = D + 4, V = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    const int4 cut = __ldcg(reinterpret_cast<const int4*>(cuts + blockIdx.x));
    const int row = blockIdx.y * 8 + warp;
    if (row >= cut.z) return;
    const float* slots = a.ws.pfx_slots + (2ll * blockIdx.x * PROWS + row) * LD;
    auto part = [&](int i) { return slots + (2ll * i + (i == 0)) * PROWS * LD; };
    float M = -INFINITY, Ls = 0.f, acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int i0 = 0; i0 < cut.w; i0 += 32) {
        const int cnt = min(32, cut.w - i0);
        const float2 ml = lane < cnt ? __ldcg(reinterpret_cast<const float2*>(part(i0 + lane))) : make_float2(-INFINITY, 0.f);
        float bm = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, o));
        const float N = fmaxf(M, bm), U = N == -INFINITY ? 0.f : N;
        const float c = exp2f(M - U), e = exp2f(ml.x - U);   // 0 for what is not there
        M = N;
        float l = ml.y * e;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        Ls = Ls * c + l;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] *= c;
#pragma unroll 1
        for (int k = 0; k < cnt; k += 4) {
            float v[4][V], w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                w[q] = __shfl_sync(0xffffffffu, e, (k + q) & 31);
#pragma unroll
                for (int i = 0; i < V; ++i) v[q][i] = 0.f;
                if (k + q < cnt) {
                    const float* p = part(i0 + k + q) + 4 + lane * V;
                    if (V == 4) {
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(p));
                        v[q][0] = x.x; v[q][1] = x.y; v[q][V - 2] = x.z; v[q][V - 1] = x.w;
                    } else {
                        const float2 x = __ldcg(reinterpret_cast<const float2*>(p));
                        v[q][0] = x.x; v[q][1] = x.y;
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] += v[q][i] * (k + q < cnt ? w[q] : 0.f);
        }
    }
    const float inv = Ls != 0.f ? 1.f / Ls : 0.f;
    const int tok = row / a.grp;
    uint16_t* out = a.out + ((long long)(cut.x + tok) * a.hq + cut.y * a.grp + row - tok * a.grp) * D;
    if (V == 4)
        *reinterpret_cast<uint2*>(out + lane * 4) =
            make_uint2(Elem<T>::pack(acc[0] * inv, acc[1] * inv), Elem<T>::pack(acc[V - 2] * inv, acc[V - 1] * inv));
    else
        *reinterpret_cast<uint32_t*>(out + lane * 2) = Elem<T>::pack(acc[0] * inv, acc[1] * inv);
}

}  // namespace paged
}  // namespace mq
