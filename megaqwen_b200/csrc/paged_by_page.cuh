// Sparse attention of many tokens, page by page: where tokens that chose the
// same page stand together, the page is read once for all of them.
//
// Mathematics: as in paged_attn.cuh, with a part (m, l, acc) for every (token,
// q head, chosen page), joined in the order of the pages.
//
// Bound: a token's chosen pages are 4 D bytes per position and kv head; with a
// few hundred tokens on one context most of that is read again and again, and
// L2 bounds it (500 tokens, 16 of 250 pages each: 2.1 GB against 134 MB that are
// distinct, 170 us).  So the choice is turned round.  The choice kernel counts
// the tokens of each (kv head, page of the pool) and notes each token's rank
// there; plan_kernel gives every page that was chosen a stretch of one list and
// cuts it into items of up to 16 query rows; list_kernel puts the tokens into
// the list; by_page_kernel walks the items, equally many to a warp.  What that
// costs are the parts, 4 (D + 4) bytes per (token, q head, page), written and
// read once, and three small launches.
//
// Measured, the same 500 tokens: clearing, plan and list 12 us together (2, 4
// and 5, mostly launch), by_page_kernel 61, join of 68 MB 16; the whole call 107
// us against 205.  by_page_kernel reads 0.33 GB (10000 items of 32 KB) and waits
// mostly for its own arithmetic: 8 warps to an SM (255 registers), each with the
// chain K Q^T, maximum, 2^x, V^T P^T per 16 positions; the tensor pipe is at
// 27 %.  Three CTAs to an SM (168 registers, spilling): 82; three ring stages
// instead of two: as fast; q rows by bulk copies instead of through L1: 112
// against 107 for the call; without the evict-first loads 38 MB of the parts
// go to HBM instead of 9.
//
// The order of a page's list depends on timing; no result does: a part's sums
// depend on its own row and the page alone (RowWarp::step with SOLO), and the
// join adds the parts in the order of the pages.
#pragma once

#include "paged_attn.cuh"

namespace mq {
namespace paged {

__global__ void __launch_bounds__(256) clear_kernel(uint4* p, long long n) {
    pdl_wait();
    pdl_trigger();
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) p[i] = make_uint4(0, 0, 0, 0);
}

// A thread to a (kv head, page); the warp takes its stretch of the list and its items by one addition to the
// cursor (items above, entries below).
__global__ void __launch_bounds__(256) plan_kernel(const ByPage w, int hkv, int pages) {
    const int lane = threadIdx.x & 31;
    const long long bin = blockIdx.x * 256ll + threadIdx.x, bins = (long long)hkv * pages;
    pdl_wait();
    pdl_trigger();
    const uint32_t cnt = bin < bins ? __ldcg(w.count + bin) : 0u;
    const uint32_t chunks = (cnt + w.per_item - 1) / (uint32_t)w.per_item;
    const unsigned long long mine = (unsigned long long)chunks << 32 | cnt;
    unsigned long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    unsigned long long base = 0;
    if (lane == 31 && x) base = atomicAdd(w.cursor, x);
    base = __shfl_sync(0xffffffffu, base, 31) + x - mine;
    const uint32_t off = (uint32_t)base, item = (uint32_t)(base >> 32);
    if (cnt) w.off[bin] = off;
    const int h = (int)(bin / pages), page = (int)(bin - (long long)h * pages);
    auto put = [&](int h, int page, uint32_t off, uint32_t cnt, uint32_t item, uint32_t i) {
        w.items[item + i] = make_int4(h, page, (int)(off + i * w.per_item), (int)min((uint32_t)w.per_item, cnt - i * w.per_item));
    };
    constexpr uint32_t OWN = 8;   // a page of more items (every token's first page, say) is the whole warp's
    if (chunks <= OWN)
        for (uint32_t i = 0; i < chunks; ++i) put(h, page, off, cnt, item, i);
    for (unsigned left = __ballot_sync(0xffffffffu, chunks > OWN); left; left &= left - 1) {
        const int src = __ffs(left) - 1;
        const uint32_t n = __shfl_sync(0xffffffffu, chunks, src), c = __shfl_sync(0xffffffffu, cnt, src);
        const uint32_t o = __shfl_sync(0xffffffffu, off, src), it = __shfl_sync(0xffffffffu, item, src);
        const int ph = __shfl_sync(0xffffffffu, h, src), pp = __shfl_sync(0xffffffffu, page, src);
        for (uint32_t i = lane; i < n; i += 32) put(ph, pp, o, c, it, i);
    }
}

// A thread to a (token, kv head, choice).
__global__ void __launch_bounds__(256) list_kernel(const RowArgs a) {
    const long long e = blockIdx.x * 256ll + threadIdx.x;
    pdl_wait();
    pdl_trigger();
    if (e >= (long long)a.total_q * a.hkv * a.top_k) return;
    const int rank = __ldcg(a.bp.rank + e);
    if (rank < 0) return;
    const uint32_t th = (uint32_t)e / (uint32_t)a.top_k, k = (uint32_t)e - th * a.top_k;   // within 31 bits
    const uint32_t t = th / (uint32_t)a.hkv, h = th - t * a.hkv;
    const int c = __ldcg(a.selected + e), pid = __ldg(a.table + __ldg(a.slots + t) * a.table_row + c);
    const uint32_t at = __ldcg(a.bp.off + (long long)h * a.pool.pages + pid) + rank;
    // how much of the page the token sees: all of it, or up to its own position
    a.bp.list[at] = make_int4((int)t, (int)k, min(__ldg(a.positions + t) + 1 - (c << a.pool.shift), a.pool.page), 0);
}

__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, int row, int h, int page, uint32_t bar,
                                              uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %2, %4, %5}], [%6], %7;"
        ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(h), "r"(page), "r"(bar), "l"(policy)
        : "memory");
}

constexpr int BY_PAGE_NT = 2;   // tiles of 8 rows to an item (one, with three CTAs to an SM: 75 us against 61)

// An item's tokens as the loading side leaves them for the computing side.
struct PageBox {
    int h, cnt, n, lim_lo;   // n: groups that any of them sees
    int4 tok[8 * BY_PAGE_NT];
};

// Loading and computing sides as in rows_kernel; an item is one page and up to
// 16 rows of the tokens that chose it.
template <typename T, int D>
__global__ void __launch_bounds__(ROW_THREADS, D == 128 ? 2 : 3)
by_page_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const RowArgs a) {
    constexpr int NT = BY_PAGE_NT;
    using W = RowWarp<T, D, NT>;
    extern __shared__ uint8_t rows_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(rows_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[ROW_WARPS][STAGES];
    // the loading side is one group ahead, so at most one item: two boxes do
    static_assert(STAGES == 2, "");
    __shared__ PageBox boxes[ROW_WARPS][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t wid = blockIdx.x * ROW_WARPS + warp, warps = gridDim.x * ROW_WARPS;
    const int grp = a.grp;
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(&full[warp][i], 1);
        fence_mbar_init();
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    __syncwarp();
    const uint64_t policy = policy_evict_first();   // pages pass through L2 once, the parts stay there for the join
    pdl_wait();
    pdl_trigger();
    const uint32_t items = (uint32_t)(__ldcg(a.bp.cursor) >> 32);
    uint32_t x = (uint32_t)((unsigned long long)items * wid / warps);
    const uint32_t xe = (uint32_t)((unsigned long long)items * (wid + 1) / warps);

    // ---- the loading side: the item after the next and the tokens of the next are on their way ----
    auto item_at = [&](uint32_t i) { return i < xe ? __ldcg(a.bp.items + i) : make_int4(0, 0, 0, 0); };
    auto tokens_of = [&](const int4& it) { return lane < it.w ? __ldcg(a.bp.list + it.z + lane) : make_int4(0, 0, 0, 0); };
    int4 it0 = item_at(x), it1 = item_at(x + 1), en = tokens_of(it0);
    int h = 0, page = 0, n = 0, k = 0, stage_l = 0, pushed = 0;
    unsigned busy = 0;   // bit i: a copy into stage i was issued and not waited for
    auto next_item = [&]() -> bool {
        if (x >= xe) return false;
        ++x;
        h = it0.x;
        page = it0.y;
        const int cnt = it0.w;
        const int hi = __reduce_max_sync(0xffffffffu, lane < cnt ? en.z : 0);
        const int lo = __reduce_min_sync(0xffffffffu, lane < cnt ? en.z : 0x7fffffff);
        n = ceil_div(hi, GRP);   // 1 or more: a token sees its own position
        k = 0;
        PageBox& b = boxes[warp][pushed & 1];
        if (lane < cnt) {
            b.tok[lane] = en;
            const uint16_t* q = a.q + (long long)en.x * a.q_tok + (long long)h * grp * a.q_head;
            for (int i = 0; i < grp; ++i, q += a.q_head) {   // its rows of q, on their way to L1
                asm volatile("prefetch.global.L1 [%0];" ::"l"(q));
                if (D == 128) asm volatile("prefetch.global.L1 [%0];" ::"l"(q + 64));
            }
        }
        if (lane == 0) {
            b.h = h;
            b.cnt = cnt;
            b.n = n;
            b.lim_lo = lo;
        }
        ++pushed;
        it0 = it1;
        it1 = item_at(x + 1);
        en = tokens_of(it0);
        return true;
    };
    W w;
    w.lane = lane;
    w.ring = smem_u32(smem) + warp * W::RING;
    auto fetch = [&]() {
        if (k < n || next_item()) {
            if (lane == 0) {
                const uint32_t bar = smem_u32(&full[warp][stage_l]), dst = w.ring + stage_l * W::STAGE;
                mbar_arrive_expect_tx(&full[warp][stage_l], W::STAGE);
                tma_load_page(dst, &tmK, k * GRP, h, page, bar, policy);
                tma_load_page(dst + W::TILE, &tmV, k * GRP, h, page, bar, policy);
            }
            busy |= 1u << stage_l;
            ++k;
        }
        stage_l = stage_l == STAGES - 1 ? 0 : stage_l + 1;
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) fetch();

    // ---- the computing side ----
    const int t = lane & 3, g = lane >> 2;
    int stage_c = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto landed = [&](int stage) -> bool {
        const long long t0 = clock64();
        bool here;
        while (!(here = mbar_try_wait(&full[warp][stage], phase >> stage & 1)) && clock64() - t0 < WAIT_CYCLES) {
        }
        phase ^= 1u << stage;
        busy &= ~(1u << stage);
        return __all_sync(0xffffffffu, here);
    };
    // which of an item's tokens this lane's rows belong to: row 8 nt + g of q, rows 8 nt + 2 t + j of the results
    int q_of[NT], r_of[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        q_of[nt] = (8 * nt + g) / grp;
        r_of[nt][0] = (8 * nt + 2 * t) / grp;
        r_of[nt][1] = (8 * nt + 2 * t + 1) / grp;
    }
    int popped = 0;
    for (; popped < pushed; ++popped) {
        __syncwarp();
        const PageBox& b = boxes[warp][popped & 1];
        const int bn = b.n, lim_lo = b.lim_lo, cnt = b.cnt;
        int lim[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int i = q_of[nt], head = b.h * grp + 8 * nt + g - i * grp;
            w.load_row(nt, i < cnt ? a.q + (long long)b.tok[i].x * a.q_tok + head * a.q_head : nullptr);
            lim[nt][0] = b.tok[min(r_of[nt][0], cnt - 1)].z;
            lim[nt][1] = b.tok[min(r_of[nt][1], cnt - 1)].z;
        }
        w.reset();
#pragma unroll 1
        for (int i = 0; i < bn; ++i) {
            fetch();
            if (!landed(stage_c)) {
                ok = false;
                break;
            }
            int rel[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                rel[nt][0] = lim[nt][0] - i * GRP;
                rel[nt][1] = lim[nt][1] - i * GRP;
            }
            w.template step<true>(stage_c, rel, lim_lo < (i + 1) * GRP, a.scale_log2);
            stage_c = stage_c == STAGES - 1 ? 0 : stage_c + 1;
            __syncwarp();   // every lane is past its reads of the stage
        }
        if (!ok) break;
        w.finish();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int i = r_of[nt][j], head = b.h * grp + 8 * nt + 2 * t + j - i * grp;
                if (i >= cnt) continue;
                const int4 tk = b.tok[i];
                w.put_part(a.bp.parts + (((long long)tk.x * a.hq + head) * a.top_k + tk.y) * W::LD, nt, j);
            }
    }
    if (!ok) {
        if (lane == 0) note_status(a.status, MQ_ERR_PIPE_TIMEOUT);
        // copies in flight land before the CTA may end
        for (int i = 0; i < STAGES; ++i)
            if (busy >> i & 1) landed(i);
    }
}

}  // namespace paged
}  // namespace mq
