// Attention over pages for few query rows: a work list of 16-position groups
// split evenly over warps, and the join of the split parts.
//
// Mathematics: softmax over j of scale q k_j, applied to v_j, by one pass with
// a running maximum m, sum l and unnormalised acc per row (log2 domain); parts
// (m, l, acc) of one row join as acc = sum acc_i 2^(m_i - M), l likewise.
//
// Bound: the keys and values are read once from HBM, 4 D bytes per position
// and kv head against 4 D flops per row.  With few rows the tensor work has to
// be small enough to hide: mma.sync m16n8k16 with the 16 positions (or 16 head
// dims) on the M side and the rows as N, so that up to 8 rows cost 8 + 16
// MMAs a group for head_dim 128 (rows on the M side cost twice that and 788
// instructions a group, and bound the kernel: 340 us for 2.1 GB from L2).
// What else has to be had is bytes in flight on every SM, whatever the
// lengths: the unit of work is one warp's 16-position group, all groups of all
// (sequence, kv head) items laid end to end and cut into equal runs, one per
// warp.  A warp keeps its own ring of TMA stages and never waits for another
// one.  A run that ends inside an item leaves a part in the workspace; the join
// kernel adds the parts in the order of the positions, so results do not
// depend on timing.
//
// Measured: 16 sequences of 64k, 2048 chosen positions each, 134 MB: 26 us (5.1
// TB/s, 0.79 of the copy rate); own parts of 64 sequences
// behind a prefix, 67 MB in 512 items: 17 us (3.9 TB/s: items of 16 groups on
// average, one or two to a warp).  From L2 it reaches 12.3 TB/s (500 tokens x 8
// kv heads x 1024 positions, 2.1 GB of which 134 MB are distinct, 170 us), which
// is why such calls go page by page (paged_by_page.cuh).
#pragma once

#include "mq_tc.cuh"
#include "paged_common.cuh"

namespace mq {
namespace paged {

constexpr int GRP = 16;            // positions per group (a page holds a whole number of them)
constexpr int MAX_RT = 16;         // query rows per item: 8 or 16
constexpr int ROW_THREADS = 128;
constexpr int ROW_WARPS = ROW_THREADS / 32;
constexpr int STAGES = 2;
constexpr int MAX_SEQS = 2048;
constexpr int MAX_TREE = 256;      // nodes of a drafted tree
constexpr int TREE_WORDS = MAX_TREE / 32;
constexpr int PK = 128;            // keys per tile and query rows per item of the tensor-core prefix kernel
constexpr int PROWS = 256;

struct PoolView {
    const uint16_t* k;   // at the layer
    const uint16_t* v;
    long long k_page, k_head, v_page, v_head;   // elements
    int pages, page, shift;   // page = 1 << shift
};

__device__ __forceinline__ int pages_for(int len, int shift) { return len <= 0 ? 0 : ((len - 1) >> shift) + 1; }

// What the join needs to know of a token: where its items start on the work
// line (kv head 0, row tile 0), how long one is, and the token's first row.
struct alignas(16) TokInfo {
    uint32_t own_base, pfx_base;
    int own_ng, own_nrt, own_r0;
    int pfx_ng, pfx_nrt, pfx_r0, pfx_rows;
    int pad[3];
};

// Part rows are m, l, pad, pad, acc[D].  A run's split item sits in slot
// 2 * worker + 1 when the run has the item's start, else in slot 2 * worker;
// a whole item with another part beside it sits at its output row.
struct WsView {
    uint32_t* head;     // [0] the call's arguments were in order, [1] units per warp, [2] units per prefix CTA
    TokInfo* tok;       // [total_q]
    float* own_rowp;    // [total_q * Hq][D + 4]
    float* slots;       // [2 * warps][rt][D + 4]
    float* pfx_rowp;    // [total_q * Hq][D + 4], twice that with the tensor-core prefix (its two streams)
    float* pfx_slots;   // [2 * CTAs][PROWS][D + 4], tensor-core prefix only
};

// Sparse attention page by page (paged_by_page.cuh).
struct ByPage {
    uint32_t* count;              // [kv heads x pages] tokens that chose the page
    unsigned long long* cursor;   // items << 32 | list entries taken
    uint32_t* off;                // [kv heads x pages] the page's place in the list
    int4* items;                  // kv head, page, place in the list, tokens
    int4* list;                   // token, choice, positions of the page that it sees
    int* rank;                    // [n, kv heads, top_k] place in the page's stretch, or -1
    float* parts;                 // [n, q heads, top_k][D + 4]
    int per_item;                 // tokens
};

struct RowArgs {
    PoolView pool;
    const uint16_t* q;
    long long q_tok, q_head;
    uint16_t* out;
    const int* table;
    long long table_row;
    int num_slots, cols;
    const int* lengths;
    const int* slots;
    const int* q_starts;
    const int* group_starts;
    const int* prefix_pages;
    const int* positions;   // sparse
    const int* selected;    // sparse
    int B, NG, total_q, hq, hkv, grp, top_k;   // grp = hq / hkv
    int rt, rt_shift;       // query rows per item of rows_kernel
    int tc;                 // prefixes run on the tensor-core kernel
    float scale_log2;
    int* status;
    WsView ws;
    ByPage bp;
    int window, sinks;      // windowed: a token sees the last `window` positions up to its own and the first `sinks`
    const int* parents;     // trees: the query tokens are nodes, a node's parent within its tree or -1
};

// A box of a page: rows from `row`, blocks of 64 channels from `block`, by a map whose base is at the layer.
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, int row, int block, int h, int page,
                                              uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(block), "r"(h), "r"(page), "r"(bar)
        : "memory");
}
__device__ __forceinline__ uint32_t movm_t(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// 2^x; 2^-inf = 0, and results below the normal numbers are 0
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr long long WAIT_CYCLES = 4000000000ll;   // bound of every wait, about two seconds
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a) : "memory");
}

// ---- the work line of an attend call --------------------------------------------------
// Entities: the groups' shared prefixes, then the sequences' own parts.  Each
// has kv heads x row tiles items; an item takes ITEM_UNITS + its 16-position
// groups (or prefix tiles) of the line, the first units standing for what an
// item costs beside them (its rows, its part).  Built by every CTA for itself
// in shared memory (a few loads per sequence; a launch of its own would cost
// more).
constexpr int ITEM_UNITS = 2;

struct Sched {
    uint32_t* off;    // [NG + B + 1] units before entity e, for one kv head
    int* len;         // [B] length of the sequence, 0 when its slot is wrong
    int* grp;         // [B] its group, or -1
    int* eff;         // [NG] shared pages read for the whole group
    int* gs;          // [NG + 1]
};
__host__ __device__ inline size_t sched_bytes(int B, int NG) {
    return ((size_t)(NG + B + 1) * 4 + (size_t)B * 8 + (size_t)(2 * NG + 1) * 4 + 15) & ~(size_t)15;
}
__device__ inline Sched sched_of(uint8_t* p, int B, int NG) {
    Sched s;
    s.off = (uint32_t*)p;
    s.len = (int*)(s.off + NG + B + 1);
    s.grp = s.len + B;
    s.eff = s.grp + B;
    s.gs = s.eff + NG;
    return s;
}

__device__ __forceinline__ int q_start(const RowArgs& a, int b) { return a.q_starts ? __ldg(a.q_starts + b) : b; }

// Sink groups of a windowed sequence, and the groups of a row tile: the window of its first row to the last row's own
// position spans at most window + (tokens of the tile) - 1 positions.
__device__ __forceinline__ int groups_of(int len) { return len > 0 ? ((len - 1) >> 4) + 1 : 0; }
__device__ __forceinline__ int sink_groups(const RowArgs& a, int len) { return min(groups_of(a.sinks), groups_of(len)); }
__device__ __forceinline__ int window_groups(const RowArgs& a, int len) {
    const int tokens = (a.rt + a.grp - 2) / a.grp + 1;   // that a tile of rt rows may touch
    return min(groups_of(len), sink_groups(a, len) + ((a.window + tokens - 2) >> 4) + 2);
}

template <bool MASK>   // MASK: of a call with a window or trees
__device__ __forceinline__ int own_groups(const RowArgs& a, const Sched& s, int b) {
    if (MASK && a.window) return window_groups(a, s.len[b]);
    const int lo = s.grp[b] >= 0 ? s.eff[s.grp[b]] << a.pool.shift : 0;
    return s.len[b] > lo ? ((s.len[b] - lo - 1) >> 4) + 1 : 0;
}
__device__ __forceinline__ int row_tiles(const RowArgs& a, int rows) { return (int)(((uint32_t)rows + a.rt - 1) >> a.rt_shift); }

// Groups (or tiles) of a prefix item and its rows, in the units of the kernel that runs it.
__device__ __forceinline__ int pfx_groups(const RowArgs& a, int eff) {
    return a.tc ? (int)((((uint32_t)eff << a.pool.shift) + PK - 1) >> 7) : eff << (a.pool.shift - 4);
}
__device__ __forceinline__ int pfx_tiles(const RowArgs& a, int rows) {
    return a.tc ? (int)(((uint32_t)rows + PROWS - 1) >> 8) : row_tiles(a, rows);
}

// Returns false (for every thread) when the starts are out of order or the
// line is longer than 2^31 units.  PFX: the prefixes alone (s.len and s.grp
// are not used).  NT threads.
template <bool PFX, int NT, bool MASK = false>
__device__ inline bool build_sched(const RowArgs& a, const Sched& s, unsigned long long* scratch /* [NT / 32] */) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    bool bad = false;
    // the first sequence's slot and length are on their way while the starts are checked
    int slot0 = -1, len0 = 0;
    if (tid < a.B) {
        slot0 = __ldg(a.slots + tid);
        if (slot0 >= 0 && slot0 < a.num_slots) len0 = __ldg(a.lengths + slot0);
    }
    if (a.NG) {   // without groups there are no arrays of them
        for (int g = tid; g <= a.NG; g += NT) {
            const int x = __ldg(a.group_starts + g);
            if (x < 0 || x > a.B) bad = true;
            s.gs[g] = x;   // used only when every start is in order
            if (g < a.NG) {
                const int members = __ldg(a.group_starts + g + 1) - x;
                if (members < 0) bad = true;
                s.eff[g] = members < 2 ? 0 : min(max(__ldg(a.prefix_pages + g), 0), a.cols);   // one alone shares nothing
            }
        }
    }
    if (a.q_starts) {
        for (int b = tid; b < a.B; b += NT)
            if (__ldg(a.q_starts + b + 1) < __ldg(a.q_starts + b)) bad = true;
        if (tid == 0 && (__ldg(a.q_starts) != 0 || __ldg(a.q_starts + a.B) != a.total_q)) bad = true;
    }
    if (__syncthreads_or(bad)) return false;
    for (int b0 = tid & ~31; b0 < a.B; b0 += NT) {   // a warp's 32 sequences together
        const int b = b0 + lane;
        const bool in = b < a.B;
        int len = 0, ql = 0, g = -1;
        if (in) {
            const int slot = b == tid ? slot0 : __ldg(a.slots + b);
            ql = q_start(a, b + 1) - q_start(a, b);
            if (slot < 0 || slot >= a.num_slots) {
                if (!PFX && blockIdx.x == 0) note_status(a.status, MQ_ERR_BAD_SLOT);
            } else {
                len = b == tid ? len0 : __ldg(a.lengths + slot);
                if (len < 0 || pages_for(len, a.pool.shift) > a.cols) {
                    if (!PFX && blockIdx.x == 0) note_status(a.status, MQ_ERR_BAD_POSITION);
                    len = 0;
                }
                if (MASK && a.parents && ql > MAX_TREE) {
                    if (!PFX && blockIdx.x == 0) note_status(a.status, MQ_ERR_INVALID_ARGUMENT);
                    len = 0;
                }
            }
            if (a.NG) {
                int lo = 0, hi = a.NG;   // the last group that starts at or before b
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (s.gs[mid] <= b) lo = mid;
                    else hi = mid;
                }
                if (s.gs[lo] <= b && b < s.gs[lo + 1]) g = lo;
            }
            if (!PFX) {
                s.len[b] = len;
                s.grp[b] = g;
            }
        }
        if (a.NG) {
            // the shared part ends where the first query token of any member stands, so all its rows
            // see all of it; one update for the warp when its sequences are of one group
            const int pages = g >= 0 && ql > 0 ? max(0, len - ql) >> a.pool.shift : 0x7fffffff;
            const int g0 = __shfl_sync(0xffffffffu, g, 0);
            const bool alone = __all_sync(0xffffffffu, g == g0 || !in);
            const int least = __reduce_min_sync(0xffffffffu, pages);
            if (alone) {
                if (lane == 0 && g0 >= 0) atomicMin(&s.eff[g0], least);
            } else if (g >= 0) {
                atomicMin(&s.eff[g], pages);
            }
        }
    }
    __syncthreads();
    const int E = a.NG + (PFX ? 0 : a.B);
    auto cost_of = [&](int e) -> unsigned long long {
        int tiles, ng;
        if (e < a.NG) {
            tiles = pfx_tiles(a, (q_start(a, s.gs[e + 1]) - q_start(a, s.gs[e])) * a.grp);
            ng = pfx_groups(a, s.eff[e]);
        } else {
            const int b = e - a.NG;
            tiles = row_tiles(a, (q_start(a, b + 1) - q_start(a, b)) * a.grp);
            ng = own_groups<MASK>(a, s, b);
        }
        return ng ? (unsigned long long)(unsigned)tiles * (unsigned)(ng + ITEM_UNITS) : 0;
    };
    auto sum_up = [&](unsigned long long x) {   // inclusive, over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    unsigned long long carry = 0;
    if (E <= 32) {   // one warp's worth
        if (warp == 0) {
            const unsigned long long cost = lane < E ? cost_of(lane) : 0, x = sum_up(cost);
            if (lane < E) s.off[lane] = (uint32_t)(x - cost);
            if (lane == 31) {
                s.off[E] = (uint32_t)x;
                scratch[0] = x;
            }
        }
        __syncthreads();
        return scratch[0] * (unsigned)a.hkv < 0x7fffffffull;
    }
    for (int e0 = 0; e0 < E; e0 += NT) {   // NT entities at a time
        const int e = e0 + tid;
        const unsigned long long cost = e < E ? cost_of(e) : 0, x = sum_up(cost);
        if (lane == 31) scratch[warp] = x;
        __syncthreads();
        unsigned long long before = carry;
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) {
            const unsigned long long v = scratch[w];
            if (w < warp) before += v;
            carry += v;
        }
        if (e < E) s.off[e] = (uint32_t)(before + x - cost);
        __syncthreads();
    }
    if (tid == 0) s.off[E] = (uint32_t)carry;
    __syncthreads();
    return carry * (unsigned)a.hkv < 0x7fffffffull;
}

// Units per worker: an equal share, but at least an item's own units and two
// groups, so that a short call is not cut into more parts than its join is worth.
__device__ __forceinline__ uint32_t quota_of(uint32_t work, uint32_t workers) {
    const uint32_t q = work / workers + (work % workers ? 1u : 0u);
    return max(q, (uint32_t)ITEM_UNITS + 2u);
}

// One warp's 16-position group step, for NT tiles of 8 query rows.
// Lane (g, t) = (lane / 4, lane % 4) works for rows 8 n + 2 t and + 1.
template <typename T, int D, int NT>
struct RowWarp {
    static constexpr int BOX = GRP * 128;             // bytes of 16 rows x 64 channels, 128-byte swizzle
    static constexpr int TILE = (D / 64) * BOX;       // a K or V group
    static constexpr int STAGE = 2 * TILE;
    static constexpr int RING = STAGES * STAGE;
    static constexpr int KS = D / 16;                 // k-steps of K Q^T, and 16-dim tiles of O^T
    static constexpr int LD = D + 4;                  // floats of a stored part row: m, l, pad, pad, acc

    uint32_t ring;     // this warp's ring, shared-memory address (1024-byte aligned)
    int lane;
    uint32_t qb[NT][KS][2];
    float o[NT][KS][4];
    float m[NT][2], l[NT][2];

    // Q^T as the B operand: row 8 n + g, dims 16 k + 2 t (+ 8)
    __device__ __forceinline__ void load_row(int n, const uint16_t* p) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                qb[n][k][i] = p ? __ldg(reinterpret_cast<const uint32_t*>(p + 16 * k + 8 * i + 2 * (lane & 3))) : 0u;
    }
    __device__ __forceinline__ void load_q(const RowArgs& a, int tok0, int h, int grp, int r0, int rows) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int i = 8 * n + (lane >> 2), r = r0 + i, tok = r / grp;
            load_row(n, i < rows ? a.q + (long long)(tok0 + tok) * a.q_tok + (h * grp + r - tok * grp) * a.q_head : nullptr);
        }
    }

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < KS; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }
    }

    // 16-byte piece c of row r of a tile
    static __device__ __forceinline__ uint32_t piece(int r, int c) {
        return (c >> 3) * BOX + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    }

    // Rows vis .. 15 of V are zeroed: stale rows must not meet the zero weights as NaN.
    __device__ __forceinline__ void clear_rows(int stage, int vis) {
        const uint32_t vs = ring + stage * STAGE + TILE;
        for (int i = vis * (D / 8) + lane; i < GRP * (D / 8); i += 32)
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(vs + piece(i / (D / 8), i % (D / 8))), "r"(0) : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the next copy into this stage
        __syncwarp();
    }

    // lim: positions of the group (below 1: none, 16 and up: all) that rows 8 n + 2 t + i see.
    // `mixed`: the rows of the tile do not all see the same positions.  SOLO: a row's sums may not depend on
    // the rows beside it, not in their last bit; `mixed`: a row does not see all positions.
    // MASK: lim is not a count but a mask of the positions.
    template <bool SOLO, bool MASK = false>
    __device__ __forceinline__ void step(int stage, const int (&lim)[NT][2], bool mixed, float scale) {
        const uint32_t ks = ring + stage * STAGE, vs = ks + TILE;
        const int g = lane >> 2, mat = lane >> 3, r8 = lane & 7;
        // Under a mask, where a few sinks may stand far above a long window, fp16 weights are held in units of 2^-14: one of 2^-25 is
        // then no subnormal number of the type, of which half would be lost.  (Sums and parts are in the same unit.)
        constexpr float UNIT = MASK && Elem<T>::MAX < 1e5f ? 16384.f : 1.f;
        auto sees = [&](int p, int lim_r) { return MASK ? (lim_r >> p & 1) != 0 : p < lim_r; };
        // S^T = K Q^T: positions g, g + 8; rows 2 t, 2 t + 1.  Even and odd k-steps in chains of their own.
        float s[NT][4], s2[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = s2[n][i] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint32_t f[4];
            ldsm4(ks + piece((mat & 1) * 8 + r8, 2 * k + (mat >> 1)), f[0], f[1], f[2], f[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) Elem<T>::mma(k & 1 ? s2[n] : s[n], f, qb[n][k][0], qb[n][k][1]);
        }
        uint32_t ph[NT][2], pr[NT][2];   // P^T as the B operand, value and remainder: positions 2 t (+ 8), row g
        bool moved = false;
        float corr[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = g + 8 * (i >> 1);
                s[n][i] = sees(p, lim[n][i & 1]) ? (s[n][i] + s2[n][i]) * scale : -INFINITY;
            }
            float u[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float mx = fmaxf(s[n][i], s[n][2 + i]);
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                const float mn = fmaxf(m[n][i], mx);
                corr[n][i] = mn == m[n][i] ? 1.f : ex2(m[n][i] - mn);   // m = -inf: nothing summed yet
                moved |= mn != m[n][i];
                m[n][i] = mn;
                u[i] = mn == -INFINITY ? 0.f : mn;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = ex2(s[n][i] - u[i & 1]) * UNIT;
            l[n][0] = l[n][0] * corr[n][0] + (s[n][0] + s[n][2]);
            l[n][1] = l[n][1] * corr[n][1] + (s[n][1] + s[n][3]);
            // two pieces of the 16-bit type: one would cost as much accuracy as rounding the output does
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t v = Elem<T>::pack(s[n][2 * i], s[n][2 * i + 1]);
                const float2 b = Elem<T>::up2(v);
                ph[n][i] = movm_t(v);
                pr[n][i] = movm_t(Elem<T>::pack(s[n][2 * i] - b.x, s[n][2 * i + 1] - b.y));
            }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    o[n][i][0] *= corr[n][0];
                    o[n][i][1] *= corr[n][1];
                    o[n][i][2] *= corr[n][0];
                    o[n][i][3] *= corr[n][1];
                }
        }
        bool slow = false;
        if (mixed) {   // a masked weight of zero must not meet an infinity or NaN
            bool odd = false;
#pragma unroll
            for (int j = 0; j < TILE / 512; ++j) {
                uint32_t w[4];
                asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(vs + (lane + 32 * j) * 16) : "memory");
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    odd |= (w[i] & Elem<T>::EXP_MASK) == Elem<T>::EXP_MASK ||
                           (w[i] >> 16 & Elem<T>::EXP_MASK) == Elem<T>::EXP_MASK;
            }
            slow = __any_sync(0xffffffffu, odd);
        }
        const int vrow = (mat >> 1) * 8 + r8;
        if (!slow) {
            // O^T += V^T P^T: dims g, g + 8 of a 16-dim tile; rows 2 t, 2 t + 1
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t f[4];
                ldsm4t(vs + piece(vrow, 2 * i + (mat & 1)), f[0], f[1], f[2], f[3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    Elem<T>::mma(o[n][i], f, ph[n][0], ph[n][1]);
                    Elem<T>::mma(o[n][i], f, pr[n][0], pr[n][1]);
                }
            }
        } else {
            if (SOLO) {   // rows that see all positions, as in any other tile
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t f[4];
                    ldsm4t(vs + piece(vrow, 2 * i + (mat & 1)), f[0], f[1], f[2], f[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float x[4] = {o[n][i][0], o[n][i][1], o[n][i][2], o[n][i][3]};
                        Elem<T>::mma(x, f, ph[n][0], ph[n][1]);
                        Elem<T>::mma(x, f, pr[n][0], pr[n][1]);
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (lim[n][c & 1] >= GRP) o[n][i][c] = x[c];
                    }
                }
            }
            // one position at a time, added only to the rows that see it
            const int t = lane & 3;
            auto takes = [&](int p, int lim_r) { return sees(p, lim_r) && !(SOLO && lim_r >= GRP); };
#pragma unroll 1
            for (int p = 0; p < GRP; ++p) {
                uint32_t keep[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)   // this lane's positions 8 i + 2 t and + 1
                    keep[i] = p == 8 * i + 2 * t ? 0xffffu : p == 8 * i + 2 * t + 1 ? 0xffff0000u : 0u;
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t f[4];
                    ldsm4t(vs + piece(vrow, 2 * i + (mat & 1)), f[0], f[1], f[2], f[3]);
                    f[0] &= keep[0];
                    f[1] &= keep[0];
                    f[2] &= keep[1];
                    f[3] &= keep[1];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float x[4] = {0.f, 0.f, 0.f, 0.f};
                        Elem<T>::mma(x, f, ph[n][0] & keep[0], ph[n][1] & keep[1]);
                        Elem<T>::mma(x, f, pr[n][0] & keep[0], pr[n][1] & keep[1]);
                        if (takes(p, lim[n][0])) {
                            o[n][i][0] += x[0];
                            o[n][i][2] += x[2];
                        }
                        if (takes(p, lim[n][1])) {
                            o[n][i][1] += x[1];
                            o[n][i][3] += x[3];
                        }
                    }
                }
            }
        }
    }

    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], x);
    }
    // Row 8 n + 2 t + i, unnormalised, to a part row; eight lanes write 32 contiguous bytes.
    __device__ __forceinline__ void put_part(float* dst, int n, int i) {
        const int g = lane >> 2;
        if (g == 0) *reinterpret_cast<float2*>(dst) = make_float2(m[n][i], l[n][i]);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            dst[4 + 16 * k + g] = o[n][k][i];
            dst[4 + 16 * k + 8 + g] = o[n][k][2 + i];
        }
    }
    __device__ __forceinline__ void put_out(uint16_t* dst, int n, int i) {
        const int g = lane >> 2;
        const float inv = l[n][i] != 0.f ? 1.f / l[n][i] : 0.f;   // a row that sees nothing is zero (NaN stays NaN)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            dst[16 * k + g] = Elem<T>::down(o[n][k][i] * inv);
            dst[16 * k + 8 + g] = Elem<T>::down(o[n][k][2 + i] * inv);
        }
    }
};

// The ancestors of node i of the tree whose first token is tok0, itself among them, as bits.  A parent that does not
// come before its child counts as none.
__device__ __forceinline__ void climb(const RowArgs& a, int tok0, int i, uint32_t* bits) {
    while (i >= 0) {
        bits[i >> 5] |= 1u << (i & 31);
        const int up = __ldg(a.parents + tok0 + i);
        if (up >= i || up < -1) note_status(a.status, MQ_ERR_INVALID_ARGUMENT);
        i = up >= i ? -1 : up;
    }
}
// 16 bits of them from bit `at` on (which may lie before the first).
__device__ __forceinline__ int ancestors(const uint32_t* bits, int at) {
    if (at < 0) return at > -16 ? (int)(bits[0] << -at & 0xffffu) : 0;
    const int w = at >> 5;
    if (w >= TREE_WORDS) return 0;
    return (int)(__funnelshift_r(bits[w], w + 1 < TREE_WORDS ? bits[w + 1] : 0u, at & 31) & 0xffffu);
}

// An item as the loading side leaves it for the computing side.
struct ItemBox {
    int tok0, h, r0, rows, first;   // rows r0 .. r0 + rows - 1 of the entity; position limit of row r: first + r / grp
    int fixed;                      // the limit of every row, or -1
    int n, flags;                   // groups of this run
};
constexpr int BOXES = 4;            // the ring spans at most STAGES items, and the one in hand
enum { BOX_START = 1, BOX_WHOLE = 2, BOX_PREFIX = 4, BOX_OTHER = 8 };

// MODE 0: attend (prefixes and own parts from the schedule).  MODE 1: sparse
// (token t's item reads the pages selected[t][h][..], top_k of them).  MODE 3:
// own parts under a mask, a sliding window with sinks or a tree of drafted tokens:
// a row's positions in a group are 16 bits (windowed: two cuts; a tree: a piece of
// the node's ancestors, walked up once for an item), and the groups that no row of
// a tile sees are not read.
//
// Each warp walks its run of the line twice at once: a loading side, STAGES - 1
// groups ahead, that finds items, looks up pages and issues copies, and a
// computing side that follows.  The loads of an item's first groups (and its q
// rows, touched into L1) are under way while the item before is computed; with
// items of a few groups each the latency would otherwise be paid per item
// (measured: 5500 cycles for an item of one group).
template <typename T, int D, int MODE, int NT>
__global__ void __launch_bounds__(ROW_THREADS, NT == 2 && D == 128 ? 2 : 3)
rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const RowArgs a) {
    using W = RowWarp<T, D, NT>;
    constexpr int RT = 8 * NT;
    extern __shared__ uint8_t rows_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(rows_raw) + 1023) & ~uintptr_t(1023));
    __shared__ unsigned long long scratch[ROW_WARPS];
    __shared__ uint64_t full[ROW_WARPS][STAGES];
    __shared__ ItemBox boxes[ROW_WARPS][BOXES];
    constexpr bool LINE = MODE == 0 || MODE == 3;
    __shared__ uint32_t above[MODE == 3 ? ROW_WARPS : 1][MODE == 3 ? RT : 1][MODE == 3 ? TREE_WORDS : 1];   // a row's ancestors
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t wid = blockIdx.x * ROW_WARPS + warp, warps = gridDim.x * ROW_WARPS;
    const int grp = a.grp, shift = a.pool.shift, page = a.pool.page;
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(&full[warp][i], 1);
        fence_mbar_init();
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    __syncwarp();
    // After a prefix kernel nothing of its is read here: it started dependents only when everything before it
    // was complete, so this kernel goes ahead beside its tail and waits for it at the end (the join needs both).
    if (MODE == 1 || !a.tc) pdl_wait();
    pdl_trigger();
    Sched s;
    uint32_t work, origin = 0;   // where this kernel's work starts on the line
    const int sp_nrt = row_tiles(a, grp), sp_ng = a.top_k << (shift - 4);
    if (LINE) {
        s = sched_of(smem + ROW_WARPS * W::RING, a.B, a.NG);
        const bool ok = build_sched<false, ROW_THREADS, MODE == 3>(a, s, scratch);
        if (!ok) {
            if (blockIdx.x == 0 && threadIdx.x == 0) {
                note_status(a.status, MQ_ERR_INVALID_ARGUMENT);
                a.ws.head[0] = 0;
            }
            if (a.tc) pdl_wait();
            return;
        }
        origin = a.tc ? s.off[a.NG] * a.hkv : 0;
        work = s.off[a.NG + a.B] * a.hkv - origin;
    } else {
        work = (uint32_t)a.total_q * a.hkv * sp_nrt * (sp_ng + ITEM_UNITS);
    }
    const uint32_t quota = quota_of(work, warps);

    // ---- the loading side ----
    uint32_t x = min(wid * quota, work);   // wid * quota < 2^32: work < 2^31, and quota is about work / warps
    const uint32_t xe = min(x + quota, work);
    int e, it, items, ng, nrt;             // entity, item in it, its items, an item's groups and row tiles
    int slot, base, tok0, rows_all, first, fixed;   // of the entity
    bool prefix = false, other = false;
    auto open = [&]() {   // entity e
        if (LINE) {
            prefix = e < a.NG;
            int b0, b1;
            first = base = 0;
            fixed = -1;
            other = false;
            if (prefix) {
                b0 = s.gs[e];
                b1 = s.gs[e + 1];
                ng = pfx_groups(a, s.eff[e]);
                fixed = ng * GRP;
            } else {
                b0 = e - a.NG;
                b1 = b0 + 1;
                ng = own_groups<MODE == 3>(a, s, b0);
                other = s.grp[b0] >= 0 && s.eff[s.grp[b0]] > 0;
                base = other ? s.eff[s.grp[b0]] << shift : 0;
            }
            tok0 = q_start(a, b0);
            const int ql = q_start(a, b1) - tok0;
            rows_all = ql * grp;
            if (!prefix) first = s.len[b0] - ql + 1;
            nrt = prefix ? pfx_tiles(a, rows_all) : row_tiles(a, rows_all);
            items = ng ? nrt * a.hkv : 0;
            if (items) {
                // a prefix is read through a member's row of the table; a member without query tokens may have none
                while (prefix && q_start(a, b0 + 1) == q_start(a, b0)) ++b0;
                slot = __ldg(a.slots + b0);
            }
        } else {
            // (kv head, token), the head outermost: tokens side by side read the same pages' rows of
            // one head, and those of one head fit L2
            tok0 = e % a.total_q;
            slot = __ldg(a.slots + tok0);
            fixed = __ldg(a.positions + tok0) + 1;
            rows_all = grp;
            ng = sp_ng;
            items = nrt = sp_nrt;
            first = base = 0;
        }
    };
    int h = 0, g0 = 0, n = 0, k = 0, lim_hi = 0;   // the item's head, its first group and groups in this run, the next one
    int lim_lo = 0, g_sink = 0, g_skip = 0;        // windowed: where its rows' windows begin, sink groups, groups left out behind them
    int ids = -1, at = 0;                          // lane i: page and position of the i-th of a batch of 32 groups
    int ring_at = -1;                              // lane i: position of the group in stage i, or -1 for nothing
    int stage_l = 0, pushed = 0;
    auto look = [&]() {
        const int kk = k + lane;
        bool want = false;
        ids = -1;
        at = 0;
        if (kk < n) {
            if (LINE) {
                at = base + (g0 + kk) * GRP;
                if (MODE == 3 && g0 + kk >= g_sink) at += g_skip * GRP;
                // past the end, or between the sinks and the windows: in no row's sight
                if (MODE == 3 && (at >= lim_hi || (at >= a.sinks && at + GRP <= lim_lo))) at = 0x7fffffff;
                else ids = __ldg(a.table + slot * a.table_row + (at >> shift));
                want = MODE != 3 || at != 0x7fffffff;
            } else {
                const int j = (g0 + kk) >> (shift - 4);
                const int c = __ldg(a.selected + ((long long)tok0 * a.hkv + h) * a.top_k + j);
                if (c >= 0) {   // listed: the slot and the column are in range
                    at = (c << shift) + (g0 + kk - (j << (shift - 4))) * GRP;
                    ids = __ldg(a.table + slot * a.table_row + c);
                    want = true;
                }
            }
            if (ids < 0 || ids >= a.pool.pages) {
                if (want) note_status(a.status, MQ_ERR_BAD_PAGE);
                ids = -1;
            }
            if (at >= lim_hi) ids = -1;   // past what any row of the tile sees
        }
    };
    // The item at x, if the run has groups of it, into the box.
    auto next_item = [&]() -> bool {
        while (x < xe) {
            while (it >= items) {
                ++e;
                it = 0;
                open();
            }
            // x lies in item `it`, which starts at x - within
            const uint32_t start = LINE ? s.off[e] * a.hkv - origin + (uint32_t)it * (ng + ITEM_UNITS)
                                             : ((uint32_t)e * items + it) * (ng + ITEM_UNITS);
            const uint32_t lo = max(x, start + ITEM_UNITS), hi = min(xe, start + ITEM_UNITS + ng);
            x = max(x, hi);
            const int i = it;
            if (hi == start + ITEM_UNITS + ng) ++it;   // done with it
            if (lo >= hi) {
                x = xe;   // the run ends in the item's own units
                return false;
            }
            h = LINE ? i / nrt : e / a.total_q;
            const int r0 = (LINE ? i - h * nrt : i) * RT, rows = min(RT, rows_all - r0);
            g0 = (int)(lo - start) - ITEM_UNITS;
            n = (int)(hi - lo);
            k = 0;
            lim_hi = fixed >= 0 ? fixed : first + (r0 + rows - 1) / grp;
            if (MODE == 3 && a.window) {
                lim_lo = first + r0 / grp - a.window;
                g_sink = min(groups_of(a.sinks), ng);
                // a tile whose groups are all of the sequence's leaves none out
                g_skip = ng == groups_of(s.len[e]) ? 0 : max(0, max(lim_lo, 0) / GRP - g_sink);
            }
            if (lane == 0) {
                ItemBox& b = boxes[warp][pushed % BOXES];
                b.tok0 = tok0;
                b.h = h;
                b.r0 = r0;
                b.rows = rows;
                b.first = first;
                b.fixed = fixed;
                b.n = n;
                b.flags = (g0 == 0 ? BOX_START : 0) | (n == ng ? BOX_WHOLE : 0) | (prefix ? BOX_PREFIX : 0) | (other ? BOX_OTHER : 0);
            }
            if (lane < rows) {
                const int r = r0 + lane;
                const uint16_t* q = a.q + (long long)(tok0 + r / grp) * a.q_tok + (h * grp + r % grp) * a.q_head;
                asm volatile("prefetch.global.L1 [%0];" ::"l"(q));
                if (D == 128) asm volatile("prefetch.global.L1 [%0];" ::"l"(q + 64));
            }
            ++pushed;
            look();
            return true;
        }
        return false;
    };

    W w;
    w.lane = lane;
    w.ring = smem_u32(smem) + warp * W::RING;
    if (x < xe) {   // where the run starts
        if (LINE) {
            const uint32_t xh = (x + origin) / (uint32_t)a.hkv;
            int lo = 0, hi = a.NG + a.B;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s.off[mid] <= xh) lo = mid;
                else hi = mid;
            }
            e = lo;
            open();
            it = (int)((x + origin - s.off[e] * a.hkv) / (uint32_t)(ng + ITEM_UNITS));
        } else {
            const uint32_t i = x / (uint32_t)(sp_ng + ITEM_UNITS);
            e = (int)(i / (uint32_t)sp_nrt);
            it = (int)(i - (uint32_t)e * sp_nrt);
            open();
        }
    }
    auto fetch = [&]() {
        int p = -1;
        if (k < n || next_item()) {
            if (k && (k & 31) == 0) look();
            const int pid = __shfl_sync(0xffffffffu, ids, k & 31), p0 = __shfl_sync(0xffffffffu, at, k & 31);
            if (pid >= 0) {
                if (lane == 0) {
                    const uint32_t bar = smem_u32(&full[warp][stage_l]), dst = w.ring + stage_l * W::STAGE;
                    mbar_arrive_expect_tx(&full[warp][stage_l], W::STAGE);
                    tma_load_page(dst, &tmK, p0 & (page - 1), 0, h, pid, bar);
                    tma_load_page(dst + W::TILE, &tmV, p0 & (page - 1), 0, h, pid, bar);
                }
                p = p0;
            }
            ++k;
        }
        if (lane == stage_l) ring_at = p;
        stage_l = stage_l == STAGES - 1 ? 0 : stage_l + 1;
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) fetch();

    // ---- the computing side ----
    const int t = lane & 3;
    int stage_c = 0;
    uint32_t phase = 0;      // bit i: parity of stage i's next copy
    bool ok = true;
    auto landed = [&](int stage) -> bool {
        const long long t0 = clock64();
        bool here;
        while (!(here = mbar_try_wait(&full[warp][stage], phase >> stage & 1)) && clock64() - t0 < WAIT_CYCLES) {
        }
        phase ^= 1u << stage;
        return __all_sync(0xffffffffu, here);
    };
    for (int popped = 0; ok && popped < pushed; ++popped) {
        __syncwarp();
        const ItemBox b = boxes[warp][popped % BOXES];
        w.load_q(a, b.tok0, b.h, grp, b.r0, b.rows);
        w.reset();
        auto limit = [&](int r) { return b.fixed >= 0 ? b.fixed : b.first + (b.r0 + min(r, b.rows - 1)) / grp; };
        const int lim_first = limit(0), lim_top = limit(b.rows - 1);
        bool walked = false;
        int lim[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) lim[n][i] = limit(8 * n + 2 * t + i);
#pragma unroll 1
        for (int i = 0; i < b.n; ++i) {
            fetch();
            const int p0 = __shfl_sync(0xffffffffu, ring_at, stage_c);
            if (p0 >= 0) {
                if (!landed(stage_c)) {
                    ok = false;
                    break;
                }
                int rel[NT][2];
                if (MODE == 3) {
                    auto low = [](int k) { return (1 << min(max(k, 0), 16)) - 1; };
                    const int base_c = b.first - 1;   // a tree's first position
                    if (a.parents && !walked && p0 + GRP > base_c) {
                        walked = true;
                        if (lane < RT) {
#pragma unroll
                            for (int i = 0; i < TREE_WORDS; ++i) above[MODE == 3 ? warp : 0][lane][i] = 0;
                            if (lane < b.rows) climb(a, b.tok0, (b.r0 + lane) / grp, above[MODE == 3 ? warp : 0][lane]);
                        }
                        __syncwarp();
                    }
                    bool full = true, none = true;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            int bits;
                            if (a.parents) {
                                bits = low(base_c - p0);
                                if (walked) {
                                    const int r = min(8 * n + 2 * t + i, b.rows - 1);
                                    bits |= ancestors(above[MODE == 3 ? warp : 0][r], p0 - base_c);
                                }
                            } else {
                                bits = low(lim[n][i] - p0);
                                bits &= ~low(lim[n][i] - a.window - p0) | low(a.sinks - p0);
                            }
                            rel[n][i] = bits;
                            full &= bits == 0xffff;
                            none &= bits == 0;
                        }
                    if (!__all_sync(0xffffffffu, none))
                        w.template step<false, true>(stage_c, rel, !__all_sync(0xffffffffu, full), a.scale_log2);
                } else {
                    if (lim_top - p0 < GRP) w.clear_rows(stage_c, lim_top - p0);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        rel[n][0] = lim[n][0] - p0;
                        rel[n][1] = lim[n][1] - p0;
                    }
                    w.template step<false>(stage_c, rel, lim_first < min(p0 + GRP, lim_top), a.scale_log2);
                }
            }
            stage_c = stage_c == STAGES - 1 ? 0 : stage_c + 1;
            __syncwarp();   // every lane is past its reads of the stage
        }
        if (!ok) break;
        w.finish();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 8 * n + 2 * t + i;
                if (r >= b.rows) continue;
                const int tk = (b.r0 + r) / grp;
                const long long row = (long long)(b.tok0 + tk) * a.hq + b.h * grp + b.r0 + r - tk * grp;
                if (!(b.flags & BOX_WHOLE))
                    w.put_part(a.ws.slots + ((2ll * wid + (b.flags & BOX_START ? 1 : 0)) * RT + r) * W::LD, n, i);
                else if (b.flags & (BOX_PREFIX | BOX_OTHER))
                    w.put_part((b.flags & BOX_PREFIX ? a.ws.pfx_rowp : a.ws.own_rowp) + row * W::LD, n, i);
                else
                    w.put_out(a.out + row * D, n, i);
            }
    }
    if (!ok) {
        if (lane == 0) note_status(a.status, MQ_ERR_PIPE_TIMEOUT);
        // copies in flight land before the CTA may end: the stages after the one that did not
        for (int i = 1; i < STAGES; ++i) {
            stage_c = stage_c == STAGES - 1 ? 0 : stage_c + 1;
            if (__shfl_sync(0xffffffffu, ring_at, stage_c) >= 0) landed(stage_c);
        }
    }
    if (LINE) {
        // the join's view of the line, a share of the sequences per warp
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            a.ws.head[0] = 1;
            a.ws.head[1] = quota;
        }
        for (int b = (int)wid; b < a.B; b += (int)warps) {
            const int q0 = q_start(a, b), q1 = q_start(a, b + 1), gr = s.grp[b];
            TokInfo ti = {};
            ti.own_base = s.off[a.NG + b] * a.hkv - origin;
            ti.own_ng = own_groups<MODE == 3>(a, s, b);
            ti.own_nrt = row_tiles(a, (q1 - q0) * grp);
            int p0 = 0;
            if (gr >= 0 && s.eff[gr] > 0) {
                p0 = q_start(a, s.gs[gr]);
                ti.pfx_base = s.off[gr] * a.hkv;
                ti.pfx_ng = pfx_groups(a, s.eff[gr]);
                ti.pfx_rows = (q_start(a, s.gs[gr + 1]) - p0) * grp;
                ti.pfx_nrt = pfx_tiles(a, ti.pfx_rows);
            }
            for (int i = q0 + lane; i < q1; i += 32) {
                ti.own_r0 = (i - q0) * grp;
                ti.pfx_r0 = (i - p0) * grp;
                a.ws.tok[i] = ti;
            }
        }
        if (a.tc) pdl_wait();
    }
}

// ---- the join ----------------------------------------------------------------------------
// acc = sum of the parts' acc_i 2^(m_i - M) over sum l_i 2^(m_i - M).  Bound by the
// latency of three dependent reads (what a token has, the parts' m and l, their acc):
// 1024 rows of 34 parts, 18 MB: 9 us; 2048 rows of 20: 9 us.
// MODE 2: sparse page by page, a part to each page that a token chose.
// SPLIT warps share a row (the fewer rows, the more parts each), 8 / SPLIT rows to a CTA.
template <typename T, int D, int MODE, int SPLIT>
__global__ void __launch_bounds__(256, 3) join_kernel(const RowArgs a, uint32_t row_warps) {
    constexpr int LD = D + 4, V = D / 32;
    __shared__ float sm_m[8], sm_l[8], sm_o[8][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long rowi = (long long)blockIdx.x * (8 / SPLIT) + warp / SPLIT;
    if (rowi >= (long long)a.total_q * a.hq) return;
    const int sub = warp % SPLIT;
    const int tok = (int)((uint32_t)rowi / (uint32_t)a.hq), head = (int)(rowi - (long long)tok * a.hq);   // rows fit 31 bits
    const int grp = a.grp, h = head / grp, RT = a.rt;
    uint16_t* out = a.out + rowi * D;
    pdl_wait();
    pdl_trigger();
    // both reads under way before either is looked at
    uint4 hd = make_uint4(0, 0, 0, 0);
    union {
        uint4 w[3];
        TokInfo ti;
    } u;
    if (MODE == 0) {
        hd = __ldcg(reinterpret_cast<const uint4*>(a.ws.head));
        const uint4* p = reinterpret_cast<const uint4*>(a.ws.tok + tok);
#pragma unroll
        for (int i = 0; i < 3; ++i) u.w[i] = __ldcg(p + i);
    }
    // the row's parts: np0 of the prefix (sub of them per run), then np1 of its own
    const float *src0 = nullptr, *src1 = nullptr;
    long long step0 = 0, step1 = 0;   // floats between parts
    int np0 = 0, np1 = 0, sub0 = 1;
    long long first0 = 0, first1 = 0, sub_step0 = 0;   // the first part of a split item is one slot further on
    if (MODE == 0) {
        if (!hd.x) {   // refused: zeros
            for (int d = sub * 32 + lane; d < D; d += SPLIT * 32) out[d] = 0;
            return;
        }
    }
    const int* there = nullptr;
    if (MODE == 2) {
        there = a.bp.rank + ((long long)tok * a.hkv + h) * a.top_k;
        src1 = a.bp.parts + rowi * a.top_k * LD;
        step1 = LD;
        np1 = a.top_k;
    }
    const int sp_ng = MODE == 1 ? a.top_k << (a.pool.shift - 4) : 0;
    const uint32_t quota =
        MODE == 0 ? hd.y
                  : quota_of((uint32_t)a.total_q * a.hkv * row_tiles(a, grp) * (sp_ng + ITEM_UNITS), row_warps);
    if (MODE != 2) {
        int ng, r;
        uint32_t start;   // the item's first group on the line
        if (MODE == 0) {
            const TokInfo& ti = u.ti;
            ng = ti.own_ng;
            r = ti.own_r0 + head % grp;
            start = ti.own_base + ((uint32_t)h * ti.own_nrt + (r >> a.rt_shift)) * (ng + ITEM_UNITS) + ITEM_UNITS;
            if (ti.pfx_ng) {
                const int R = a.tc ? PROWS : RT, pr = ti.pfx_r0 + head % grp, in = pr & (R - 1);
                const uint32_t ps = ti.pfx_base + ((uint32_t)h * ti.pfx_nrt + (uint32_t)(pr - in) / R) * (ti.pfx_ng + ITEM_UNITS) + ITEM_UNITS;
                const uint32_t pq = a.tc ? hd.z : quota, w0 = ps / pq;
                const int runs = (int)((ps + ti.pfx_ng - 1) / pq - w0) + 1;
                if (a.tc && min(PROWS, ti.pfx_rows - (pr - in)) <= 128) sub0 = 2;   // both streams worked on this row
                np0 = runs * sub0;
                if (runs == 1) {
                    src0 = a.ws.pfx_rowp + rowi * LD;
                    sub_step0 = (long long)a.total_q * a.hq * LD;
                } else {
                    src0 = (a.tc ? a.ws.pfx_slots : a.ws.slots) + (2ll * w0 * R + in) * LD;
                    step0 = 2ll * R * LD;
                    first0 = (long long)R * LD;
                    sub_step0 = 128ll * LD;
                }
            }
        } else {
            const int nrt = row_tiles(a, grp);
            r = head % grp;
            ng = sp_ng;
            start = (((uint32_t)h * a.total_q + tok) * nrt + (r >> a.rt_shift)) * (ng + ITEM_UNITS) + ITEM_UNITS;
        }
        if (ng) {
            const uint32_t w0 = start / quota;
            np1 = (int)((start + ng - 1) / quota - w0) + 1;
            if (np1 == 1) {
                if (!np0) return;   // written by the only warp that had it
                src1 = a.ws.own_rowp + rowi * LD;
            } else {
                src1 = a.ws.slots + (2ll * w0 * RT + (r & (RT - 1))) * LD;
                step1 = 2ll * RT * LD;
                first1 = (long long)RT * LD;
            }
        }
    }
    auto part = [&](int i) -> const float* {
        if (i < np0) {
            const int j = i / sub0;
            return src0 + j * step0 + (j == 0 ? first0 : 0) + (i - j * sub0) * sub_step0;
        }
        i -= np0;
        return src1 + i * step1 + (i == 0 ? first1 : 0);
    };
    const int np = np0 + np1;
    // A batch of 32 parts at a time: lane i finds part i and its maximum and sum (one round
    // trip), then the rows of acc are read eight in flight, whatever their weights are.
    float M = -INFINITY, L = 0.f, acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int i0 = sub; i0 < np; i0 += SPLIT * 32) {
        const int mine = i0 + SPLIT * lane, cnt = min(32, (np - i0 + SPLIT - 1) / SPLIT);
        const float* p = mine < np ? part(mine) : nullptr;
        const int at = MODE == 2 && mine < np ? __ldcg(there + mine) : 0;
        float2 ml = p ? __ldcg(reinterpret_cast<const float2*>(p)) : make_float2(-INFINITY, 0.f);
        if (at < 0) {   // nothing was written there
            p = nullptr;
            ml = make_float2(-INFINITY, 0.f);
        }
        float bm = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, o));
        const float N = fmaxf(M, bm), U = N == -INFINITY ? 0.f : N;
        const float c = exp2f(M - U), e = exp2f(ml.x - U);   // 0 for what is not there
        M = N;
        float l = ml.y * e;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        L = L * c + l;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] *= c;
#pragma unroll 1
        for (int k = 0; k < cnt; k += 8) {
            float v[8][V], w[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float* r = reinterpret_cast<const float*>(
                    __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), (k + q) & 31));
                w[q] = __shfl_sync(0xffffffffu, e, (k + q) & 31);
#pragma unroll
                for (int i = 0; i < V; ++i) v[q][i] = 0.f;
                if (k + q < cnt && (MODE != 2 || r)) {
                    if (V == 4) {
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(r + 4) + lane);
                        v[q][0] = x.x; v[q][1] = x.y; v[q][V - 2] = x.z; v[q][V - 1] = x.w;
                    } else {
                        const float2 x = __ldcg(reinterpret_cast<const float2*>(r + 4) + lane);
                        v[q][0] = x.x; v[q][1] = x.y;
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < 8; ++q)
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] += v[q][i] * (k + q < cnt ? w[q] : 0.f);
        }
    }
    if (SPLIT > 1) {
        if (lane == 0) {
            sm_m[warp] = M;
            sm_l[warp] = L;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sm_o[warp][lane * V + i] = acc[i];
        named_bar_sync(1 + warp / SPLIT, SPLIT * 32);   // the row's warps (all or none of them got here)
        if (sub) return;
        float MM = -INFINITY;
#pragma unroll
        for (int k = 0; k < SPLIT; ++k) MM = fmaxf(MM, sm_m[warp + k]);
        const float UU = MM == -INFINITY ? 0.f : MM;
        L = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
        for (int k = 0; k < SPLIT; ++k) {
            const float e = exp2f(sm_m[warp + k] - UU);
            L += sm_l[warp + k] * e;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += sm_o[warp + k][lane * V + i] * e;
        }
    }
    const float inv = L != 0.f ? 1.f / L : 0.f;
    if (V == 4)
        *reinterpret_cast<uint2*>(out + lane * 4) =
            make_uint2(Elem<T>::pack(acc[0] * inv, acc[1] * inv), Elem<T>::pack(acc[V - 2] * inv, acc[V - 1] * inv));
    else
        *reinterpret_cast<uint32_t*>(out + lane * 2) = Elem<T>::pack(acc[0] * inv, acc[1] * inv);
}

}  // namespace paged
}  // namespace mq
