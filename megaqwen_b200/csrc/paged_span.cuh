// Attention under a mask for many query rows, on the 5th-generation tensor
// cores: sliding windows with sinks, trees of drafted tokens.
//
// Work: items of (sequence, kv head, up to 256 query rows: whole tokens) x the
// 128-key tiles that any of its rows sees, a windowed item's sink tiles first.
// Items lie end to end on a line that is cut into equal runs, one per CTA (one
// CTA per SM), each item as long as it has tiles.
//
// A CTA runs two streams, A and B, as the shared-prefix kernel does
// (paged_prefix.cuh): with more than 128 rows each has half of them and every tile
// is used by both; with up to 128 rows both take the same ones, A the even tiles
// and B the odd, and their two accumulators, side by side in TMEM, are joined when
// the item ends.  Weights go into the second product as two 16-bit pieces.
//
// Masks: a tile that some row does not see whole has its scores set to minus
// infinity in TMEM by two cuts (windowed) or by the node's ancestors (a tree),
// whose tiles are few; other tiles take no test.  An infinity or NaN among values
// that a row does not see must not meet its zero weight: a warp of its own looks
// through the masked tiles' values, puts zeros in their place and notes where they
// were, and a row that does see one has a NaN in that channel at the end.
//
// An item that a run's end cuts leaves a part (m, l, acc) per row and run, which
// the join adds in the order of the positions.
#pragma once

#include "paged_prefix.cuh"

namespace mq {
namespace paged {

constexpr int SPAN_THREADS = 384;   // warps: 0 items and K, 1 MMA, 2 Q and V, 3 looks through V, 4-7 softmax of A, 8-11 of B
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
    static constexpr int SCHED = ODD + 2 * 128 * (D / 8);
    static constexpr size_t bytes(int B) { return SCHED + (size_t)(2 * B + 1) * 4 + 1024; }
};

// An item that is cut: the worker with its first tile leaves this for the join.
struct alignas(16) SpanCut {
    int tok0, h, rows, runs;   // rows 0: none
};

struct alignas(16) SpanSeg {
    int slot, h, tok0, rows;      // tok0: the tile's first token; rows: of this item
    int seq0, pf, pl;             // the sequence's first token; positions of the tile's first and last token
    int st, wt, ng;               // sink tiles, first window tile, tiles in all
    int t0, n, runs;              // of this run (n 0: the run is over); runs that share the item
    bool two, both, start, whole;   // two: each stream has rows of its own; both: B works, too
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
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 128 consecutive columns of this warp's TMEM lanes, waited for.
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, float* v) {
    uint32_t r[128];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x128.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,"
        "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
        "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
        "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"
        "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%128];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
          "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
          "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]),
          "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]),
          "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]),
          "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]),
          "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]),
          "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]),
          "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 128; ++i) v[i] = __uint_as_float(r[i]);
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
    uint64_t* s_full = bars + 12;     // [2] streams: S is there (and every MMA issued before it is done)
    uint64_t* p_full = bars + 14;     // [2] P is stored, O is rescaled
    uint64_t* o_full = bars + 16;     // [2] the run's last PV is done
    uint64_t* q_empty = bars + 18;    // [2]
    uint64_t* drain = bars + 20;
    uint64_t* pair = bars + 21;       // [4] the warps of A and B on the same rows
    uint64_t* item_full = bars + 25;  // [SPAN_ITEMS]
    uint64_t* item_empty = item_full + SPAN_ITEMS;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(item_empty + SPAN_ITEMS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
    volatile int* holes = abort_flag + 1;      // a page out of range has been met
    volatile int* odd_tile = abort_flag + 2;   // [2] stages: the tile holds values that are not finite
    __shared__ uint32_t scratch[NT / 32];
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&v_ready[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(drain, 1);
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
    int* lens = reinterpret_cast<int*>(off + a.B + 1);              // [B], 0 where nothing is read
    const int grp = a.grp, page = a.pool.page, tps = PROWS / 2 / grp, tpt = 2 * tps;   // tokens to a stream and to a row tile
    bool bad = false;
    if (a.q_starts) {
        for (int b = threadIdx.x; b < a.B; b += NT)
            if (__ldg(a.q_starts + b + 1) < __ldg(a.q_starts + b)) bad = true;
        if (threadIdx.x == 0 && (__ldg(a.q_starts) != 0 || __ldg(a.q_starts + a.B) != a.total_q)) bad = true;
    }
    bool in_order = !__syncthreads_or(bad);
    {
        unsigned long long carry = 0;
        for (int b0 = 0; in_order && b0 < a.B; b0 += NT) {
            const int b = b0 + threadIdx.x;
            unsigned long long cost = 0;
            if (b < a.B) {
                const int slot = __ldg(a.slots + b), ql = q_start(a, b + 1) - q_start(a, b);
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
                    if (blockIdx.x == 0) note_status(a.status, code);
                }
                lens[b] = len;
                int st, wt;
                for (int i = 0; len && i < ql; i += tpt) {
                    const int n = span_tiles(a, len - ql + i, len - ql + min(i + tpt, ql) - 1, st, wt);
                    cost += n ? n + ITEM_UNITS : 0;
                }
            }
            unsigned long long x = cost;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const bool big = x > 0x7fffffffull;   // a sum that does not fit is refused below
            if (lane == 31) scratch[warp] = big ? 0x7fffffffu : (uint32_t)x;
            __syncthreads();
            unsigned long long before = carry;
            for (int w = 0; w < NT / 32; ++w) {
                const uint32_t v = scratch[w];
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

    // The item at x and the tiles of it in this run (n <= 0: the run has only its own units); x moves past them.
    // By the first warp.
    auto segment = [&](uint32_t& x) {
        SpanSeg e;
        const uint32_t xh = x / (uint32_t)a.hkv;
        int lo = 0, hi = a.B;   // the last sequence that starts at or before, of those with work
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (off[mid] <= xh) lo = mid;
            else hi = mid;
        }
        e.slot = __ldg(a.slots + lo);
        const uint32_t one = off[lo + 1] - off[lo];
        uint32_t rel = x - off[lo] * a.hkv;
        e.h = (int)(rel / one);
        rel -= e.h * one;
        e.seq0 = q_start(a, lo);
        const int ql = q_start(a, lo + 1) - e.seq0, p0 = lens[lo] - ql;
        for (int i0 = 0;; i0 += 32) {   // the row tile, 32 at a time
            const int i = (i0 + lane) * tpt;
            int st, wt, n = 0;
            if (i < ql) n = span_tiles(a, p0 + i, p0 + min(i + tpt, ql) - 1, st, wt);
            const uint32_t cost = n ? n + ITEM_UNITS : 0;
            uint32_t sum = cost;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += y;
            }
            const unsigned found = __ballot_sync(0xffffffffu, rel < sum);
            if (!found && (i0 + 32) * tpt < ql) {
                rel -= __shfl_sync(0xffffffffu, sum, 31);
                continue;
            }
            const int at = found ? __ffs((int)found) - 1 : 0;   // (always found: x is within the sequence)
            rel -= __shfl_sync(0xffffffffu, sum - cost, at);
            const int first = (i0 + at) * tpt, last = min(first + tpt, ql) - 1;
            e.tok0 = e.seq0 + first;
            e.rows = (last - first + 1) * grp;
            e.pf = p0 + first;
            e.pl = p0 + last;
            break;
        }
        e.ng = span_tiles(a, e.pf, e.pl, e.st, e.wt);
        const int pos = (int)rel, left = (int)min((uint32_t)(e.ng + ITEM_UNITS - pos), xe - x);
        e.t0 = max(pos - ITEM_UNITS, 0);
        e.n = max(pos + left - ITEM_UNITS, 0) - e.t0;
        e.two = e.rows > tps * grp;
        e.both = e.two || e.n > 1;
        e.start = e.t0 == 0;
        e.whole = e.n == e.ng;
        const uint32_t ps = x - pos + ITEM_UNITS;   // the item's first tile on the line
        e.runs = (int)((ps + e.ng - 1) / quota - ps / quota) + 1;
        x += left;
        return e;
    };
    auto tile_at = [&](const SpanSeg& e, int j) {   // first position of the run's j-th tile
        const int t = e.t0 + j;
        return (t < e.st ? t : e.wt + t - e.st) * PK;
    };
    // Every row sees all of the tile at `at`.
    auto all_seen = [&](const SpanSeg& e, int at) {
        if (a.parents) return at + PK <= e.seq0 - e.tok0 + e.pf;
        return at + PK - 1 <= e.pf && (at > e.pl - a.window || at + PK <= a.sinks);
    };
    // Some row sees a position of the page at `at`: other pages' entries in the table are not looked at.
    auto in_sight = [&](const SpanSeg& e, int at) {
        return at <= e.pl && (a.parents || at < a.sinks || at + page > e.pf - a.window + 1);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
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

    if (warp == 0 || warp == 2) {
        // ---- K and V producers: lane c loads the tile's c-th page.  That of V also loads the items' Q, a box of whole
        // tokens for each stream, once the last scores of the item before are there ----
        uint64_t* full = warp == 0 ? k_full : v_full;
        uint64_t* empty = warp == 0 ? k_empty : v_empty;
        const CUtensorMap* map = warp == 0 ? &tmK : &tmV;
        uint8_t* ring = smem + (warp == 0 ? L::K : L::V);
        const int chunks = PK / page;
        int c = 0, nq0 = 0, nq1 = 0;   // tiles so far, Q tiles of A and B
        bool ok = true, cut = false;
        auto load_q = [&](const SpanSeg& e, int q, int used) {
            if (used && !wait(&q_empty[q], (used - 1) & 1)) return false;
            if (lane == 0) {
                mbar_arrive_expect_tx(&q_full[q], (D / 64) * tps * grp * 128);
#pragma unroll
                for (int i = 0; i < D / 64; ++i)
                    tma_load_heads(smem_u32(smem + L::Q + q * TILE + i * PATOM), &tmQ, i, e.h * grp,
                                   e.tok0 + (e.two ? q * tps : 0), smem_u32(&q_full[q]));
            }
            return true;
        };
        uint32_t x = x0;
        SpanSeg e;
        while (ok) {
            if (warp == 0) {
                e.n = 0;
                while (x < xe && e.n <= 0) e = segment(x);
                if (taken >= SPAN_ITEMS)
                    ok = __all_sync(0xffffffffu, wait(&item_empty[taken % SPAN_ITEMS], (taken / SPAN_ITEMS - 1) & 1));
                if (!ok) break;
                if (lane == 0) {
                    item_at(taken) = e;
                    mbar_arrive(&item_full[taken % SPAN_ITEMS]);
                }
                ++taken;
                if (e.n <= 0) break;
                if (e.start && !e.whole) {   // (the run's last item)
                    if (lane == 0) *reinterpret_cast<int4*>(cuts + blockIdx.x) = make_int4(e.tok0, e.h, e.rows, e.runs);
                    cut = true;
                }
            } else {
                if (!take(e, ok)) break;
                done_with();
                ok = load_q(e, 0, nq0++);
                if (ok && e.both) ok = load_q(e, 1, nq1++);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
            }
            const int* row = a.table + e.slot * a.table_row;
            // what no row sees is read as zeros, from outside the map
            auto look = [&](int j) {
                const int at = tile_at(e, j) + lane * page;
                return lane < chunks && in_sight(e, at) ? __ldg(row + (at >> a.pool.shift)) : a.pool.pages;
            };
            int next = look(0);
            for (int j = 0; j < e.n; ++j, ++c) {
                int pid = next;
                if (j + 1 < e.n) next = look(j + 1);
                if (pid < 0 || pid >= a.pool.pages) {
                    if (lane < chunks && in_sight(e, tile_at(e, j) + lane * page)) {
                        note_status(a.status, MQ_ERR_BAD_PAGE);
                        *holes = 1;   // before the tile's scores are there
                    }
                    pid = a.pool.pages;
                }
                const int st = c & 1;
                const bool here = c < 2 || wait(&empty[st], ((c >> 1) - 1) & 1);
                if (!__all_sync(0xffffffffu, here)) {
                    ok = false;
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(&full[st], TILE);
                __syncwarp();
                if (lane < chunks) {
#pragma unroll
                    for (int i = 0; i < D / 64; ++i)
                        tma_load_page(smem_u32(ring + st * TILE + i * PATOM + lane * page * 128), map, 0, i, e.h, pid, smem_u32(&full[st]));
                }
            }
        }
        if (warp == 0 && !cut && lane == 0) *reinterpret_cast<int4*>(cuts + blockIdx.x) = make_int4(0, 0, 0, 0);
        if (!ok && lane == 0) give_up();
        // copies in flight land before the CTA may end, whatever became of their readers
        auto land = [&](uint64_t* bar, uint32_t parity) {
            const long long t0 = clock64();
            while (!mbar_try_wait(bar, parity) && clock64() - t0 < WAIT_CYCLES) {
            }
        };
        for (int k = max(0, c - 2); k < c; ++k) land(&full[k & 1], (k >> 1) & 1);
        if (!ok && warp == 2) {   // (otherwise the scores of every Q tile have been waited for)
            if (nq0) land(&q_full[0], (nq0 - 1) & 1);
            if (nq1) land(&q_full[1], (nq1 - 1) & 1);
        }
    } else if (warp == 3) {
        // ---- looks through the values of masked tiles ----
        int c = 0;
        bool ok = true;
        for (SpanSeg e; take(e, ok); done_with()) {
            for (int j = 0; j < e.n; ++j, ++c) {
                const int st = c & 1;
                ok = __all_sync(0xffffffffu, wait(&v_full[st], (c >> 1) & 1));
                if (!ok) break;
                if (!all_seen(e, tile_at(e, j))) {
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
            }
        }
        if (!ok && lane == 0) give_up();
    } else if (warp == 1) {
        // ---- MMA: the whole warp walks, one elected lane issues.  All 512 columns of
        // TMEM are this CTA's, so their addresses start at 0 ----
        constexpr uint32_t id_o = pfx_idesc<T>(D, true);
        // a negative scale: the scores of -Q
        const uint32_t id_s = pfx_idesc<T>(PK, false) | (a.scale_log2 < 0.f ? 1u << 13 : 0u);
        const uint32_t base = (smem_u32(pfx_raw) + 1023u) & ~1023u;
        int c0 = 0;                         // tiles of the segments before
        uint32_t np0 = 0, np1 = 0;          // PVs issued per stream
        uint32_t nq0 = 0, nq1 = 0;          // Q tiles used per stream
        bool ok = true;
        auto scores = [&](int q, int kc, bool last_use, bool last) {
            const uint32_t sq = base + L::Q + q * TILE, sk = base + L::K + (kc & 1) * TILE;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint32_t o = (k >> 2) * PATOM + (k & 3) * 32;
                tc_mma_f16(q * 128, sw128_kmajor_desc(sq + o), sw128_kmajor_desc(sk + o), id_s, k != 0);
            }
            tc_commit(&s_full[q]);
            if (last_use) tc_commit(&k_empty[kc & 1]);
            if (last) tc_commit(&q_empty[q]);
        };
        auto values = [&](int q, int vc, bool first, bool last_use, bool done) {
            const uint32_t sv = base + L::V + (vc & 1) * TILE, o = 256 + q * 128;
#pragma unroll
            for (int k = 0; k < PK / 16; ++k) {
                const uint32_t p = q * 128 + 8 * k;   // 16 keys: 8 columns
                tc_mma_f16_ts(o, p, sw128_mnmajor_desc(sv + k * 2048), id_o, !first || k);
            }
            if (last_use) tc_commit(&v_empty[vc & 1]);
            if (done) tc_commit(&o_full[q]);
        };
        for (SpanSeg e; take(e, ok); done_with()) {
            const int n = uniform(e.n);
            const bool two = uniform(e.two);
            const int steps = two ? 2 * n : n;
            // step i: the stream's PV of its tile before (step i - 2), then its S of this one.  What the
            // step needs is waited for by four lanes at once.
            for (int i = 0; ok && i < steps + 2; ++i) {
                const int q = i & 1;
                const bool pv = i >= 2, sc = i < steps;
                const int vc = c0 + (two ? (i - 2) >> 1 : i - 2), kc = c0 + (two ? i >> 1 : i);
                if (!pv && !sc) continue;   // a run of one tile: stream B has none
                uint64_t* bar = nullptr;
                uint32_t parity = 0;
                if (lane == 0 && sc) bar = &k_full[kc & 1], parity = kc >> 1;
                if (lane == 1 && pv) bar = &v_ready[vc & 1], parity = vc >> 1;
                if (lane == 2 && pv) bar = &p_full[q], parity = q ? np1 : np0;
                if (lane == 3 && !pv) bar = &q_full[q], parity = q ? nq1 : nq0;
                ok = __all_sync(0xffffffffu, !bar || wait(bar, parity & 1));
                if (pv) (q ? np1 : np0)++;
                else (q ? nq1 : nq0)++;
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    if (pv) values(q, vc, i < 4, !two || q == 1, !sc);
                    if (sc) scores(q, kc, !two || q == 1, i >= steps - 2);
                }
                __syncwarp();
            }
            c0 += n;
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
        ulonglong2* hits = reinterpret_cast<ulonglong2*>(smem + L::HIT);
        constexpr float GROW = 8.f;
        int ns = 0, nv = 0, no0 = 0, no1 = 0, np = 0;   // scores taken, tiles of the items before, results of A and B, meetings
        bool ok = true;
        auto got = [&](uint64_t* bar, uint32_t parity) {
            if (ok) ok = __all_sync(0xffffffffu, wait(bar, parity));
            return ok;
        };
        auto meet = [&]() {   // with the other stream's warp on the same rows
            __syncwarp();
            if (lane == 0) mbar_arrive(&pair[quad]);
            got(&pair[quad], np++ & 1);
        };
        const int tok_r = r / grp, head_r = r - tok_r * grp;   // of this row in its stream
        for (SpanSeg e; take(e, ok); done_with()) {
            const int mine = e.two ? e.n : (e.n + 1 - q) >> 1;   // this stream's tiles
            const int tok = (e.two ? q * tps : 0) + tok_r;       // the row's token in the item
            const bool there = tok_r < tps && tok * grp < e.rows;
            const int pos = min(e.pf + tok, e.pl), node = e.tok0 - e.seq0 + pos - e.pf;
            unsigned long long hit[2] = {0, 0};
            float m = -INFINITY, l = 0.f;
#pragma unroll 1
            for (int j = 0; j < mine; ++j, ++ns) {
                const int jt = e.two ? j : 2 * j + q, at = tile_at(e, jt);
                const bool masked = !all_seen(e, at);
                unsigned long long live[2] = {~0ull, ~0ull};   // keys that the row sees
                if (masked) {
                    live[0] = span_sees(a, pos, at, node, e.seq0);
                    live[1] = span_sees(a, pos, at + 64, node, e.seq0);
                }
                if (!got(&s_full[q], ns & 1)) break;
                tc_fence_after();
                if (*holes) {   // pages out of range: their keys are left out
                    const int* row = a.table + e.slot * a.table_row;
                    for (int k = 0; k < PK; k += min(page, 64)) {
                        const int p = (at + k) & -page;
                        const int pid = in_sight(e, p) ? __ldg(row + (p >> a.pool.shift)) : 0;
                        if (pid < 0 || pid >= a.pool.pages) {
                            const unsigned long long gone = ~((page >= 64 ? ~0ull : (1ull << page) - 1ull) << (k & 63));
                            if (k < 64) live[0] &= gone;
                            else live[1] &= gone;
                        }
                    }
                }
                float sv[128], mx[4];
                tmem_ld128(sa, sv);
                if (__any_sync(0xffffffffu, (live[0] & live[1]) != ~0ull)) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t b = (uint32_t)(live[w >> 1] >> (32 * (w & 1)));
#pragma unroll
                        for (int k = 0; k < 32; ++k) sv[32 * w + k] = b >> k & 1u ? sv[32 * w + k] : -INFINITY;
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) mx[k] = fmaxf(sv[2 * k], sv[2 * k + 1]);
#pragma unroll
                for (int k = 8; k < 128; k += 2) mx[(k >> 1) & 3] = max3(mx[(k >> 1) & 3], sv[k], sv[k + 1]);
                const float tmax = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * scale;
                // a row's maximum moves only when it grew by more than 2^8; weights stay below 256
                float corr = 1.f;
                if (tmax > m + GROW) {
                    corr = ex2(m - tmax);   // 0 on the first tile
                    m = tmax;
                }
                l *= corr;
                if (j && __any_sync(0xffffffffu, corr != 1.f)) {
                    // s_full covers the PV before it, so O is at rest
#pragma unroll 1
                    for (int i = 0; i < D; i += 16) {
                        float v[16];
                        tmem_ld16(oa + q * 128 + i, v);
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[k] *= corr;
                        tmem_st16(oa + q * 128 + i, v);
                    }
                }
                const uint64_t scale2 = two_of(scale, scale), u2 = m == -INFINITY ? 0ull : two_of(-m, -m);
                uint64_t sum0 = 0ull, sum1 = 0ull;
#pragma unroll
                for (int i = 0; i < 128; i += 32) {
                    uint32_t pk[16];   // 32 weights in 16 columns, over the scores
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float p0, p1;
                        halves(fma2(two_of(sv[i + 2 * k], sv[i + 2 * k + 1]), scale2, u2), p0, p1);
                        p0 = ex2(p0);
                        p1 = ex2(p1);
                        (k & 1 ? sum1 : sum0) = add2(k & 1 ? sum1 : sum0, two_of(p0, p1));
                        pk[k] = Elem<T>::pack(p0, p1);
                    }
                    tmem_st16_nowait(sa + (i >> 1), pk);
                }
                float s0, s1;
                halves(add2(sum0, sum1), s0, s1);
                l += s0 + s1;
                if (masked) {
                    // the tile's values are looked through, and stay until this stream's weights are used
                    const int c = nv + jt, st = c & 1;
                    if (got(&v_ready[st], (c >> 1) & 1) && odd_tile[st]) {
                        const uint8_t* bits = smem + L::ODD + st * 128 * (D / 8);
#pragma unroll 1
                        for (int k = 0; k < PK; ++k) {
                            if (!((k < 64 ? live[0] : live[1]) >> (k & 63) & 1ull)) continue;
                            hit[0] |= *reinterpret_cast<const unsigned long long*>(bits + k * (D / 8));
                            if (D == 128) hit[1] |= *reinterpret_cast<const unsigned long long*>(bits + k * (D / 8) + 8 * (D / 128));
                        }
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[q]);
            }
            nv += e.n;
            // ---- the item's rows: what A and B have of them, when they share them ----
            if (!e.two || q == 0) got(&o_full[0], no0 & 1);
            if (e.two ? q == 1 : e.both) got(&o_full[1], no1 & 1);
            ++no0;
            no1 += e.both;
            tc_fence_after();
            float e0 = 1.f, e1 = 1.f;   // weights of A's and B's accumulators
            if (!e.two) {
                sums[q * 128 + r] = l;
                tops[q * 128 + r] = m;
                hits[q * 128 + r] = make_ulonglong2(hit[0], hit[1]);
                meet();
                const float ma = tops[r], mb = tops[128 + r];   // (B's is -inf when it had no tile)
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
            float* part = there ? a.ws.pfx_slots + ((2ll * blockIdx.x + e.start) * PROWS + tok * grp + head_r) * LD : nullptr;
            uint16_t* out = there ? a.out + ((long long)(e.tok0 + tok) * a.hq + e.h * grp + head_r) * D : nullptr;
            if (!e.whole && ok && there && (e.two || q == 0)) *reinterpret_cast<float4*>(part) = make_float4(m, l, 0.f, 0.f);
#pragma unroll 1
            for (int c = c_lo; ok && c < c_hi; c += 32) {
                float v[32];
                tmem_ld32(oa + (e.two ? q * 128 : 0) + c, v);
                if (!e.two) {
                    float w[32];
                    if (e.both) tmem_ld32(oa + 128 + c, w);
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = e.both ? v[k] * e0 + w[k] * e1 : v[k] * e0;
                }
                const uint32_t odd = (uint32_t)(hit[c >> 6] >> (c & 63));
                if (odd) {
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (odd >> k & 1u) v[k] = NAN;
                }
                if (!e.whole) {
                    if (there) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            *reinterpret_cast<float4*>(part + 4 + c + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                    }
                    continue;
                }
                // four pieces of 16 bytes; four lanes turn theirs into whole 64 bytes of their four rows, so that a
                // store touches eight rows and not 32
                uint32_t w[4][4];
#pragma unroll
                for (int k = 0; k < 16; ++k) w[k >> 2][k & 3] = Elem<T>::pack(v[2 * k] * inv, v[2 * k + 1] * inv);
#pragma unroll
                for (int x = 1; x < 4; x <<= 1) {
                    const bool high = lane & x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i & x) continue;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t other = __shfl_xor_sync(0xffffffffu, high ? w[i][k] : w[i | x][k], x);
                            (high ? w[i][k] : w[i | x][k]) = other;
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint16_t* to = from_lane(out, (lane & ~3) + k);
                    if (to) *reinterpret_cast<uint4*>(to + c + (lane & 3) * 8) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
                }
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
                const int t0 = q_start(a, b), ql = q_start(a, b + 1) - t0;
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

// The join of the items that were cut: acc = sum acc_i 2^(m_i - M) over sum l_i 2^(m_i - M).  blockIdx.y: a CTA's rows of
// the cut; a warp to a row.
constexpr int SPAN_JOIN_ROWS = 8;
template <typename T, int D>
__global__ void __launch_bounds__(256) span_join_kernel(const RowArgs a, const SpanCut* __restrict__ cuts) {
    constexpr int LD = D + 4, V = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    const int4 cut = __ldcg(reinterpret_cast<const int4*>(cuts + blockIdx.x));
    const int row = blockIdx.y * SPAN_JOIN_ROWS + warp;
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
