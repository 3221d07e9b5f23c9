// Pages of the paged KV cache: reserve, fork, free, copy, compact.
//
// Bookkeeping is exact and independent of scheduling: pages are handed out
// lowest number first, in the order of the caller's list, so two runs give the
// same tables.  Each operation that needs a decision over all pages makes it
// in one CTA ("plan": validation, a scan of the counts, a list of moves in the
// workspace), and a second, wide kernel carries it out; plan and move are
// chained by programmatic dependent launch.  A plan that finds its arguments, or the
// rows that they name, wrong writes the status word and a move count of zero, and
// nothing changes; free and reserve alike.
//
// Bound: HBM for the moves, a page's rows read and written once by warps of 16-byte
// accesses, eight in flight.  153 pages of 28 layers (1.14 GB both ways) into
// another pool: 181 us, 6.3 TB/s, 0.96 of the copy rate; 64 copies of 40 rows of
// one page (294 MB written, 4.6 MB read): 50 us, 5.9 TB/s.  Latency for the plans, free and
// reserve: 4 to 7 us each, a dozen dependent reads of one CTA.
#include <algorithm>

#include "paged_common.cuh"

namespace mq {
namespace paged {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_WARPS = PLAN_THREADS / 32;
constexpr int MAX_SLOTS = 65536;
constexpr int MAX_PAGES = 1 << 20;   // a plan's sums of 1024 counts of up to MAX_PAGES + 1 stay below 2^31
constexpr int MOVE_THREADS = 256;

// Workspace: a header, then the lists of a plan.
struct Plan {
    int* head;    // [0] moves, [1] plan accepted
    int* src;     // [cap] page read
    int* dst;     // [cap] page written (-1: none)
    int* rows;    // [cap] rows moved
    int* ids;     // [num_pages] pages found by a scan, ascending
    int* map;     // [num_pages] old page -> new page
    int* off;     // [n + 1] exclusive sums
    unsigned* bits;   // [num_pages / 32 + 1]
};

size_t plan_ints(int num_pages, int n) {
    const size_t cap = (size_t)std::max(num_pages, n);
    return 16 + 3 * cap + 2 * (size_t)num_pages + (size_t)n + 1 + (size_t)num_pages / 32 + 1;
}

Plan plan_of(void* ws, int num_pages, int n) {
    const size_t cap = (size_t)std::max(num_pages, n);
    Plan p;
    p.head = (int*)ws;
    p.src = p.head + 16;
    p.dst = p.src + cap;
    p.rows = p.dst + cap;
    p.ids = p.rows + cap;
    p.map = p.ids + num_pages;
    p.off = p.map + num_pages;
    p.bits = (unsigned*)(p.off + n + 1);
    return p;
}

struct Tab {
    int* table;
    int* lengths;
    int* refs;
    int slots, cols, pages, page;
    long long row;
    int* status;
};

Tab tab_of(const mq_page_table* t) {
    return {t->table, t->lengths, t->refs, t->num_slots, t->cols, t->num_pages, t->page_size, t->row_stride, t->status};
}

// ---- scans by one CTA of 1024 threads ---------------------------------------------

// Exclusive sum of one value per thread; *total gets the sum.  Ends with every
// thread past its reads of the scratch.
__device__ int block_scan(int v, int* sm, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) sm[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = sm[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        sm[lane] = w;
    }
    __syncthreads();
    const int base = warp ? sm[warp - 1] : 0;
    *total = sm[PLAN_WARPS - 1];
    __syncthreads();
    return base + x - v;
}

// Pages with refs > 0 (live) or == 0 (free), in ascending order: ids[r] = the
// r-th, for r < limit; map[p] = r or -1, if given.  Returns how many there are.
// Each warp counts a contiguous segment by ballots, one block scan places the
// segments, and a second pass (the counts come from L1 / L2) writes them: two
// passes over 4 bytes a page cost less than a block-wide scan per 1024 pages.
__device__ int find_pages(const int* refs, int P, bool live, int* ids, int limit, int* map, int* sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int seg = (ceil_div(P, PLAN_WARPS) + 31) & ~31;
    const int lo = min(P, warp * seg), hi = min(P, lo + seg);
    int count = 0;
#pragma unroll 4
    for (int i = lo; i < hi; i += 32) {
        const int p = i + lane;
        const int r = p < hi ? refs[p] : -1;
        count += __popc(__ballot_sync(0xffffffffu, p < hi && (live ? r > 0 : r == 0)));
    }
    int total;
    // one value per warp: the other lanes add nothing
    int at = block_scan(lane == 0 ? count : 0, sm, &total);
    at = __shfl_sync(0xffffffffu, at, 0);
#pragma unroll 4
    for (int i = lo; i < hi; i += 32) {
        const int p = i + lane;
        const int r = p < hi ? refs[p] : -1;
        const bool yes = p < hi && (live ? r > 0 : r == 0);
        const unsigned m = __ballot_sync(0xffffffffu, yes);
        const int rank = at + __popc(m & ((1u << lane) - 1u));
        if (yes && rank < limit) ids[rank] = p;
        if (map && p < hi) map[p] = yes ? rank : -1;
        at += __popc(m);
    }
    __syncthreads();
    return total;
}

// Every slot of the list in range and named once; leaves the set in `bits`
// (MAX_SLOTS / 32 words).  Every thread gets the answer.
__device__ bool slots_ok(const int* slots, int n, int num_slots, unsigned* bits) {
    for (int i = threadIdx.x; i < ceil_div(num_slots, 32); i += blockDim.x) bits[i] = 0;
    __syncthreads();
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = slots[i];
        if (s < 0 || s >= num_slots) bad = true;
        else if (atomicOr(&bits[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) bad = true;
    }
    return !__syncthreads_or(bad);
}

// Short lists of a plan stay in shared memory: a search through them in global
// memory was half of a reservation's time.
constexpr int NEAR_OFF = 1024, NEAR_IDS = 2048;

// ---- free ----------------------------------------------------------------------------
// One cluster over all entries of the list's rows.  The counts are taken down first;
// where one of them was not there to take (a page out of range, not in use, or held by
// more of the rows than its count says), every count is put back and nothing else is
// written.  Each CTA checks the list of slots itself (it is short).
__global__ void __launch_bounds__(PLAN_THREADS) free_kernel(Tab t, const int* __restrict__ slots, int n) {
    __shared__ unsigned bits[MAX_SLOTS / 32];
    __shared__ int wrong;
    pdl_wait();
    pdl_trigger();
    const int ranks = (int)cluster_size(), rank = (int)cluster_rank();   // (the grid is one cluster)
    // a warp to a sequence; its first row is on its way to L1 while the list is checked
    const int per = blockDim.x / 32, lane = threadIdx.x & 31, warp = rank * per + (threadIdx.x >> 5), warps = ranks * per;
    if (threadIdx.x == 0) wrong = 0;
    if (warp < n) {
        const int s = slots[warp];
        if (s >= 0 && s < t.slots) {
            asm volatile("prefetch.global.L1 [%0];" ::"l"(t.lengths + s));
            if (lane < t.cols) asm volatile("prefetch.global.L1 [%0];" ::"l"(t.table + s * t.row + lane));
        }
    }
    if (!slots_ok(slots, n, t.slots, bits)) {   // all CTAs alike
        if (rank == 0 && threadIdx.x == 0) note_status(t.status, MQ_ERR_BAD_SLOT);
        return;
    }
    if (ranks > 1) cluster_sync();   // every CTA runs and has its `wrong`: it may be written
    bool bad = false;
    for (int i = warp; i < n; i += warps) {
        const int s = slots[i], used = min(pages_of(t.lengths[s], t.page), t.cols);
        const int* row = t.table + s * t.row;
#pragma unroll 4
        for (int c = lane; c < used; c += 32) {
            const int p = row[c];
            if (p < 0 || p >= t.pages || atomicSub(&t.refs[p], 1) <= 0) bad = true;
        }
    }
    bad = __syncthreads_or(bad);
    if (ranks > 1) {
        if (bad && threadIdx.x == 0)
            for (int r = 0; r < ranks; ++r) st_peer(smem_u32(&wrong), r, 1u);
        __syncwarp();
        cluster_sync();   // also orders the counts taken before those put back
        bad = *(volatile int*)&wrong;
    }
    if (bad) {
        if (rank == 0 && threadIdx.x == 0) note_status(t.status, MQ_ERR_BAD_PAGE);
        for (int i = warp; i < n; i += warps) {
            const int s = slots[i], used = min(pages_of(t.lengths[s], t.page), t.cols);
            for (int c = lane; c < used; c += 32) {
                const int p = t.table[s * t.row + c];
                if (p >= 0 && p < t.pages) atomicAdd(&t.refs[p], 1);
            }
        }
        return;
    }
    for (int i = warp; i < n; i += warps) {
        const int s = slots[i];
        for (int c = lane; c < t.cols; c += 32) t.table[s * t.row + c] = -1;
        if (lane == 0) t.lengths[s] = 0;
    }
}

// ---- reserve -------------------------------------------------------------------------
__global__ void __launch_bounds__(PLAN_THREADS) reserve_kernel(Tab t, const int* __restrict__ slots,
                                                               const int* __restrict__ new_lengths, int n, Plan pl) {
    __shared__ unsigned bits[MAX_SLOTS / 32];
    __shared__ int sm[PLAN_WARPS], near_off[NEAR_OFF], near_ids[NEAR_IDS];
    pdl_wait();
    pdl_trigger();
    if (!slots_ok(slots, n, t.slots, bits)) {
        if (threadIdx.x == 0) note_status(t.status, MQ_ERR_BAD_SLOT);
        return;
    }
    int* off = n <= NEAR_OFF ? near_off : pl.off;
    int need = 0;
    bool bad = false;
    for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
        const int i = i0 + threadIdx.x;
        int k = 0;
        if (i < n) {
            const int have = t.lengths[slots[i]], want = new_lengths[i];
            if (have < 0 || want < have || pages_of(want, t.page) > t.cols) bad = true;
            // one sequence cannot need more than the pool has; the cap keeps the sums below 2^31
            else k = min(pages_of(want, t.page) - pages_of(have, t.page), t.pages + 1);
        }
        int sum;
        const int at = block_scan(k, sm, &sum);
        if (i < n) off[i] = need + at;
        need = min(need + sum, t.pages + 1);
        if (need > t.pages) break;
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) note_status(t.status, MQ_ERR_BAD_POSITION);
        return;
    }
    int* ids = need <= NEAR_IDS ? near_ids : pl.ids;
    if (need > 0 && (need > t.pages || find_pages(t.refs, t.pages, false, ids, need, nullptr, sm) < need)) {
        if (threadIdx.x == 0) note_status(t.status, MQ_ERR_NO_PAGES);
        return;
    }
    __syncthreads();
    for (int r = threadIdx.x; r < need; r += PLAN_THREADS) {
        int lo = 0, hi = n;   // the last sequence whose pages start at or before r
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (off[mid] <= r) lo = mid;
            else hi = mid;
        }
        const int s = slots[lo], p = ids[r];
        t.table[s * t.row + pages_of(t.lengths[s], t.page) + r - off[lo]] = p;
        t.refs[p] = 1;
    }
    __syncthreads();   // the old lengths are read above
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS) t.lengths[slots[i]] = new_lengths[i];
}

// ---- moving pages -------------------------------------------------------------------
struct Side {
    char* base;
    long long page, layer, head;   // bytes
};
struct Geo {
    Side src[3], dst[3];   // K, V, index (base null: none)
    int layers, heads, row_bytes, record;
};

Side side_of(void* base, long long page, long long layer, long long head, int bytes) {
    return {(char*)base, page * bytes, layer * bytes, head * bytes};
}

Geo geo_of(const mq_paged_pool* s, const mq_paged_pool* d, bool index) {
    Geo g;
    g.src[0] = side_of(s->k, s->k_page, s->k_layer, s->k_head, 2);
    g.src[1] = side_of(s->v, s->v_page, s->v_layer, s->v_head, 2);
    g.dst[0] = side_of(d->k, d->k_page, d->k_layer, d->k_head, 2);
    g.dst[1] = side_of(d->v, d->v_page, d->v_layer, d->v_head, 2);
    const bool ix = index && s->index && d->index;
    g.src[2] = side_of(ix ? s->index : nullptr, s->i_page, s->i_layer, s->i_head, 1);
    g.dst[2] = side_of(ix ? d->index : nullptr, d->i_page, d->i_layer, d->i_head, 1);
    g.layers = s->num_layers;
    g.heads = s->num_kv_heads;
    g.row_bytes = s->head_dim * 2;
    g.record = 2 * s->head_dim + 16;
    return g;
}

// How the pages of `b` lie on those of `a`, when both may be views of one storage: apart; a page p of `a` on page
// p + *shift of `b` alone; or tangled (any other way, or not to be told).  The [page, head_dim] blocks of one side do
// not overlap each other.
enum Lie { APART, SHIFTED, TANGLED };
Lie lie_of(const Side& a, int na, const Side& b, int nb, int layers, int heads, long long block, long long* shift) {
    if (!a.base || !b.base) return APART;
    const auto end = [&](const Side& s, int n, bool high) {   // the lowest byte, or the one after the highest
        long long at = reinterpret_cast<long long>(s.base) + (high ? block : 0);
        for (const long long x : {(n - 1) * s.page, (layers - 1) * s.layer, (heads - 1) * s.head})
            if (high ? x > 0 : x < 0) at += x;
        return at;
    };
    if (end(a, na, true) <= end(b, nb, false) || end(b, nb, true) <= end(a, na, false)) return APART;
    const long long page = nb > 1 ? b.page : a.page;
    if ((na > 1 && nb > 1 && a.page != b.page) || (layers > 1 && a.layer != b.layer) || (heads > 1 && a.head != b.head) ||
        ((na > 1 || nb > 1) && page < block))
        return TANGLED;
    if (a.base == b.base) {
        *shift = 0;
        return SHIFTED;
    }
    if ((2ll * layers - 1) * (2ll * heads - 1) > 1 << 20) return TANGLED;
    bool found = false;
    for (int l = 1 - layers; l < layers; ++l)
        for (int h = 1 - heads; h < heads; ++h) {
            // a block of b less one of a: off + d pages, for d pages between them
            const long long off = (b.base - a.base) + l * a.layer + h * a.head;
            const long long d0 = na > 1 || nb > 1 ? -off / page : 0;
            for (long long d = d0 - 1; d <= d0 + 1; ++d) {
                const long long apart = off + d * page;
                if (d <= -na || d >= nb || apart >= block || apart <= -block) continue;
                if (found && *shift != d) return TANGLED;
                found = true;
                *shift = d;
            }
        }
    return found ? SHIFTED : APART;
}

// The same for two pools: every tensor of one against those of the other.
Lie lie_of(const Geo& g, int na, int nb, int page, long long* shift) {
    const bool same = g.src[0].base == g.dst[0].base && g.src[1].base == g.dst[1].base;
    bool found = false;
    for (int i = 0; i < 3; ++i)
        for (int j = 0; j < 3; ++j) {
            if ((i == 2) != (j == 2) || (same && i != j)) continue;
            long long d = 0;
            const Lie lie = lie_of(g.src[i], na, g.dst[j], nb, g.layers, g.heads, i == 2 ? g.record : (long long)page * g.row_bytes, &d);
            if (lie == TANGLED || (lie == SHIFTED && found && d != *shift)) return TANGLED;
            if (lie == SHIFTED) {
                found = true;
                *shift = d;
            }
        }
    return found ? SHIFTED : APART;
}

// Copies `bytes` (a multiple of 16) by one warp, eight 16-byte pieces in flight per lane.
__device__ __forceinline__ void warp_copy(char* __restrict__ d, const char* __restrict__ s, int bytes, int lane) {
    int i = lane * 16;
    for (; i + 7 * 512 < bytes; i += 8 * 512) {
        uint4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const uint4*>(s + i + k * 512);
#pragma unroll
        for (int k = 0; k < 8; ++k) *reinterpret_cast<uint4*>(d + i + k * 512) = v[k];
    }
    for (; i < bytes; i += 512) *reinterpret_cast<uint4*>(d + i) = *reinterpret_cast<const uint4*>(s + i);
}

// The blocks of a plan's moves: a unit is one (move, tensor, layer, head), its
// rows contiguous on both sides, copied by one warp.  `wid` of `nw` warps.
__device__ void move_units(const Geo& g, const Plan& pl, int moves, long long wid, long long nw, int lane) {
    const int per = g.layers * g.heads, kinds = g.src[2].base ? 3 : 2;
    const long long total = (long long)moves * kinds * per;
    for (long long u = wid; u < total; u += nw) {
        const int m = (int)(u / (kinds * per)), r = (int)(u - (long long)m * kinds * per);
        const int kind = r / per, lh = r - kind * per, l = lh / g.heads, h = lh - l * g.heads;
        const int dst = pl.dst[m];
        if (dst < 0) continue;
        const Side &a = g.src[kind], &b = g.dst[kind];
        const char* s = a.base + pl.src[m] * a.page + l * a.layer + h * a.head;
        char* d = b.base + dst * b.page + l * b.layer + h * b.head;
        warp_copy(d, s, kind == 2 ? g.record : pl.rows[m] * g.row_bytes, lane);
    }
}

// ---- fork ----------------------------------------------------------------------------
__global__ void __launch_bounds__(PLAN_THREADS) fork_plan_kernel(Tab t, const int* __restrict__ parents,
                                                                 const int* __restrict__ children, int n, Plan pl) {
    __shared__ unsigned bits[MAX_SLOTS / 32], looked[MAX_SLOTS / 32];
    __shared__ int sm[PLAN_WARPS], near_off[NEAR_OFF], near_ids[NEAR_IDS];
    pdl_wait();
    pdl_trigger();
    if (threadIdx.x == 0) pl.head[1] = 0;
    for (int i = threadIdx.x; i < ceil_div(t.slots, 32); i += PLAN_THREADS) looked[i] = 0;   // (slots_ok synchronises)
    int* off = n <= NEAR_OFF ? near_off : pl.off;
    bool bad = !slots_ok(children, n, t.slots, bits);
    if (!bad) {   // the same for every thread
        for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
            const int p = parents[i];
            // a child is empty, and no parent is a child too
            if (t.lengths[children[i]] != 0 || p < 0 || p >= t.slots || (bits[p >> 5] >> (p & 31) & 1u)) bad = true;
        }
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) note_status(t.status, MQ_ERR_BAD_SLOT);
        return;
    }
    int copies = 0, wrong = 0;
    // every full page of every parent in range and in use; a warp to a parent, and each parent once
    // (from the last warp down, so that a short list's first warp goes on to the part pages meanwhile)
    for (int i = PLAN_WARPS - 1 - (threadIdx.x >> 5); i < n; i += PLAN_WARPS) {
        const int lane = threadIdx.x & 31, p = parents[i];
        int first = 0;
        if (lane == 0) first = !(atomicOr(&looked[p >> 5], 1u << (p & 31)) >> (p & 31) & 1u);
        if (!__shfl_sync(0xffffffffu, first, 0)) continue;
        const int full = min(t.lengths[p] / t.page, t.cols);   // (a length beyond the row is refused below)
#pragma unroll 4
        for (int c = lane; c < full; c += 32) {
            const int g = t.table[p * t.row + c];
            if (g < 0 || g >= t.pages || t.refs[g] <= 0) wrong |= 2;
        }
    }
    for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
        const int i = i0 + threadIdx.x;
        int part = 0, src = -1;
        if (i < n) {
            const int len = t.lengths[parents[i]];
            if (len < 0 || pages_of(len, t.page) > t.cols) {
                wrong |= 1;
            } else {
                part = len % t.page;
                if (part) {
                    src = t.table[parents[i] * t.row + len / t.page];
                    if (src < 0 || src >= t.pages || t.refs[src] <= 0) wrong |= 2;
                }
            }
        }
        int sum;
        const int at = block_scan(part > 0, sm, &sum);
        if (i < n) {
            pl.src[i] = src;
            pl.rows[i] = part;
            off[i] = part > 0 ? copies + at : -1;
        }
        copies += sum;
    }
    const int any1 = __syncthreads_or(wrong & 1), any2 = __syncthreads_or(wrong & 2);
    if (any1 || any2) {
        if (threadIdx.x == 0) note_status(t.status, any1 ? MQ_ERR_BAD_POSITION : MQ_ERR_BAD_PAGE);
        return;
    }
    int* ids = copies <= NEAR_IDS ? near_ids : pl.ids;
    if (copies > 0 && find_pages(t.refs, t.pages, false, ids, copies, nullptr, sm) < copies) {
        if (threadIdx.x == 0) note_status(t.status, MQ_ERR_NO_PAGES);
        return;
    }
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS) pl.dst[i] = off[i] >= 0 ? ids[off[i]] : -1;
    if (threadIdx.x == 0) pl.head[1] = 1;
}

__global__ void __launch_bounds__(MOVE_THREADS) fork_move_kernel(Geo g, Tab t, const int* __restrict__ parents,
                                                                 const int* __restrict__ children, int n, Plan pl) {
    pdl_wait();
    pdl_trigger();
    if (!pl.head[1]) return;
    const long long tid = (long long)blockIdx.x * MOVE_THREADS + threadIdx.x, nt = (long long)gridDim.x * MOVE_THREADS;
    for (long long e = tid; e < (long long)n * t.cols; e += nt) {
        const int i = (int)(e / t.cols), c = (int)(e - (long long)i * t.cols);
        const int par = parents[i], kid = children[i];
        const int len = t.lengths[par], full = len / t.page, dst = pl.dst[i];
        int p = -1;
        if (c < full) {
            p = t.table[par * t.row + c];   // in range: the plan looked at it
            atomicAdd(&t.refs[p], 1);
        } else if (c == full && dst >= 0) {
            p = dst;
            t.refs[p] = 1;
        }
        t.table[kid * t.row + c] = p;
        if (c == 0) t.lengths[kid] = len;
    }
    move_units(g, pl, n, tid >> 5, nt >> 5, threadIdx.x & 31);
}

// ---- copy ----------------------------------------------------------------------------
// `shared`: page p read is page p + shift written, where that is one of the dst_pages.
__global__ void __launch_bounds__(PLAN_THREADS) copy_plan_kernel(const int* __restrict__ src, const int* __restrict__ dst,
                                                                 int n, int src_pages, int dst_pages, bool shared,
                                                                 long long shift, int page, int* status, Plan pl) {
    pdl_wait();
    pdl_trigger();
    if (threadIdx.x == 0) pl.head[1] = 0;
    for (int i = threadIdx.x; i < dst_pages / 32 + 1; i += PLAN_THREADS) pl.bits[i] = 0;
    __syncthreads();
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
        const int s = src[i], d = dst[i];
        if (s < 0 || s >= src_pages || d < 0 || d >= dst_pages) bad = true;
        else if (atomicOr(&pl.bits[d >> 5], 1u << (d & 31)) >> (d & 31) & 1u) bad = true;
        pl.src[i] = s;
        pl.dst[i] = d;
        pl.rows[i] = page;
    }
    bad = __syncthreads_or(bad);
    if (!bad && shared)
        for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
            const long long d = src[i] + shift;
            if (d >= 0 && d < dst_pages && __ldcg(&pl.bits[d >> 5]) >> (d & 31) & 1u) bad = true;
        }
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
        if (bad) note_status(status, MQ_ERR_BAD_PAGE);
        pl.head[0] = n;
        pl.head[1] = !bad;
    }
}

__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(Geo g, Plan pl) {
    pdl_wait();
    pdl_trigger();
    if (!pl.head[1]) return;
    const long long tid = (long long)blockIdx.x * MOVE_THREADS + threadIdx.x, nt = (long long)gridDim.x * MOVE_THREADS;
    move_units(g, pl, pl.head[0], tid >> 5, nt >> 5, threadIdx.x & 31);
}

// ---- compact -------------------------------------------------------------------------
__global__ void __launch_bounds__(PLAN_THREADS) compact_plan_kernel(Tab t, int dst_pages, Plan pl) {
    __shared__ int sm[PLAN_WARPS];
    pdl_wait();
    pdl_trigger();
    const int live = find_pages(t.refs, t.pages, true, pl.src, t.pages, pl.map, sm);
    const bool ok = live <= dst_pages;
    for (int i = threadIdx.x; i < live; i += PLAN_THREADS) {
        pl.dst[i] = i;
        pl.rows[i] = t.page;
    }
    if (threadIdx.x == 0) {
        if (!ok) note_status(t.status, MQ_ERR_NO_PAGES);
        pl.head[0] = live;
        pl.head[1] = ok;
    }
}

__global__ void __launch_bounds__(MOVE_THREADS) compact_move_kernel(Geo g, Tab t, int dst_pages, int* __restrict__ out_table,
                                                                    long long out_row, int* __restrict__ out_refs, Plan pl) {
    pdl_wait();
    pdl_trigger();
    if (!pl.head[1]) return;
    const int live = pl.head[0];
    const long long tid = (long long)blockIdx.x * MOVE_THREADS + threadIdx.x, nt = (long long)gridDim.x * MOVE_THREADS;
    for (long long e = tid; e < (long long)t.slots * t.cols; e += nt) {
        const int s = (int)(e / t.cols), c = (int)(e - (long long)s * t.cols);
        const int p = t.table[s * t.row + c];
        out_table[s * out_row + c] = p >= 0 && p < t.pages ? pl.map[p] : -1;
    }
    for (long long i = tid; i < dst_pages; i += nt) out_refs[i] = i < live ? t.refs[pl.src[i]] : 0;
    move_units(g, pl, live, tid >> 5, nt >> 5, threadIdx.x & 31);
}

bool tab_ok(const mq_page_table* t, int n, bool lengths) {
    return t && t->table && (t->lengths || !lengths) && t->refs && t->num_slots >= 1 && t->num_slots <= MAX_SLOTS &&
           t->cols >= 1 && t->num_pages >= 1 && t->num_pages <= MAX_PAGES && t->row_stride >= t->cols && n >= 0 && n <= t->num_slots &&
           (t->page_size == 16 || t->page_size == 32 || t->page_size == 64 || t->page_size == 128);
}

bool same_geometry(const mq_paged_pool* a, const mq_paged_pool* b) {
    return a->dtype == b->dtype && a->num_layers == b->num_layers && a->num_kv_heads == b->num_kv_heads &&
           a->page_size == b->page_size && a->head_dim == b->head_dim && !a->index == !b->index;
}

int done(cudaError_t e, const char* what) { return e == cudaSuccess ? MQ_OK : note_cuda(e, what); }

int move_grid() { return sm_count() * 8; }

}  // namespace paged
}  // namespace mq

using namespace mq::paged;

extern "C" {

size_t mq_paged_workspace_bytes(int num_pages, int n) {
    if (num_pages < 0 || n < 0) return 0;
    return plan_ints(num_pages, n) * sizeof(int);
}

int mq_paged_free(const mq_page_table* t, const int* slots, int n, cudaStream_t st) {
    if (!tab_ok(t, n, true) || (n && !slots)) return MQ_ERR_INVALID_ARGUMENT;
    if (!n) return MQ_OK;
    if (n <= 8) return done(launch(free_kernel, dim3(1), dim3(256), 0, st, tab_of(t), slots, n), "paged free");
    unsigned ranks = 1;   // a warp to a sequence; 64 sequences take the same time with 1, 2 and 8 CTAs
    while (ranks < 8 && (int)ranks * PLAN_WARPS < n) ranks *= 2;
    return done(launch_cluster(free_kernel, ranks, ranks, dim3(PLAN_THREADS), 0, st, tab_of(t), slots, n), "paged free");
}

int mq_paged_reserve(const mq_page_table* t, const int* slots, const int* new_lengths, int n, cudaStream_t st) {
    if (!tab_ok(t, n, true) || (n && (!slots || !new_lengths))) return MQ_ERR_INVALID_ARGUMENT;
    if (!n) return MQ_OK;
    if (!t->workspace || t->workspace_bytes < mq_paged_workspace_bytes(t->num_pages, n)) return MQ_ERR_WORKSPACE;
    return done(launch(reserve_kernel, dim3(1), dim3(PLAN_THREADS), 0, st, tab_of(t), slots, new_lengths, n,
                       plan_of(t->workspace, t->num_pages, n)), "paged reserve");
}

int mq_paged_fork(const mq_paged_pool* pool, const mq_page_table* t, const int* parents, const int* children, int n,
                  cudaStream_t st) {
    if (!pool_ok(pool) || !tab_ok(t, n, true) || (n && (!parents || !children)) || pool->num_pages != t->num_pages ||
        pool->page_size != t->page_size)
        return MQ_ERR_INVALID_ARGUMENT;
    if (!n) return MQ_OK;
    if (!t->workspace || t->workspace_bytes < mq_paged_workspace_bytes(t->num_pages, n)) return MQ_ERR_WORKSPACE;
    const Plan pl = plan_of(t->workspace, t->num_pages, n);
    cudaError_t e = launch(fork_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, st, tab_of(t), parents, children, n, pl);
    if (e == cudaSuccess)
        e = launch(fork_move_kernel, dim3(move_grid()), dim3(MOVE_THREADS), 0, st, geo_of(pool, pool, false), tab_of(t),
                   parents, children, n, pl);
    return done(e, "paged fork");
}

int mq_paged_copy(const mq_paged_pool* src, const mq_paged_pool* dst, const int* src_pages, const int* dst_pages, int n,
                  int* status, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    if (!pool_ok(src) || !pool_ok(dst) || !same_geometry(src, dst) || n < 0 || (n && (!src_pages || !dst_pages)))
        return MQ_ERR_INVALID_ARGUMENT;
    const Geo g = geo_of(src, dst, true);
    long long shift = 0;
    const Lie lie = lie_of(g, src->num_pages, dst->num_pages, src->page_size, &shift);
    if (lie == TANGLED) return MQ_ERR_INVALID_ARGUMENT;
    if (!n) return MQ_OK;
    if (!workspace || workspace_bytes < mq_paged_workspace_bytes(dst->num_pages, n)) return MQ_ERR_WORKSPACE;
    const Plan pl = plan_of(workspace, dst->num_pages, n);
    cudaError_t e = launch(copy_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, st, src_pages, dst_pages, n, src->num_pages,
                           dst->num_pages, lie == SHIFTED, shift, src->page_size, status, pl);
    if (e == cudaSuccess) e = launch(move_kernel, dim3(move_grid()), dim3(MOVE_THREADS), 0, st, g, pl);
    return done(e, "paged copy");
}

int mq_paged_compact(const mq_paged_pool* src, const mq_paged_pool* dst, const mq_page_table* t, int* out_table,
                     long long out_row_stride, int* out_refs, cudaStream_t st) {
    if (!pool_ok(src) || !pool_ok(dst) || !same_geometry(src, dst) || !tab_ok(t, 0, false) || !out_table || !out_refs ||
        src->num_pages != t->num_pages || src->page_size != t->page_size || out_row_stride < t->cols ||
        out_table == t->table || out_refs == t->refs)
        return MQ_ERR_INVALID_ARGUMENT;
    const Geo g = geo_of(src, dst, true);
    long long shift = 0;
    if (lie_of(g, src->num_pages, dst->num_pages, src->page_size, &shift) != APART) return MQ_ERR_INVALID_ARGUMENT;
    if (!t->workspace || t->workspace_bytes < mq_paged_workspace_bytes(t->num_pages, 0)) return MQ_ERR_WORKSPACE;
    const Plan pl = plan_of(t->workspace, t->num_pages, 0);
    cudaError_t e = launch(compact_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, st, tab_of(t), dst->num_pages, pl);
    if (e == cudaSuccess)
        e = launch(compact_move_kernel, dim3(move_grid()), dim3(MOVE_THREADS), 0, st, g, tab_of(t),
                   dst->num_pages, out_table, out_row_stride, out_refs, pl);
    return done(e, "paged compact");
}

}  // extern "C"
