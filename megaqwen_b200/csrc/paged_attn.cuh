// Attention over pages for few query rows: a work list of 16-position groups
// split evenly over warps, and the join of the split parts.
//
// Mathematics: softmax over j of scale q k_j, applied to v_j, by one pass with
// a running maximum m, sum l and unnormalised acc per row (log2 domain); parts
// (m, l, acc) of one row join as acc = sum acc_i 2^(m_i - M), l likewise.
//
// Bound: the keys and values are read once from HBM, 4 D bytes per position
// and kv head against 4 D flops per row, so with up to 16 rows the tensor work
// (mma.sync m16n8k16, rows on the M side) hides behind the loads.  What has to
// be had is bytes in flight on every SM, whatever the lengths: the unit of
// work is one warp's 16-position group, all groups of all (sequence, kv head)
// items laid end to end and cut into equal runs, one per warp.  A warp keeps
// its own ring of cp.async stages and never waits for another one.  A run that
// ends inside an item leaves a part in the workspace; the join kernel adds the
// parts in the order of the positions, so results do not depend on timing.
#pragma once

#include "paged_common.cuh"

namespace mq {
namespace paged {

constexpr int GRP = 16;            // positions per group (a page holds a whole number of them)
constexpr int RT = 16;             // query rows per item
constexpr int ROW_THREADS = 128;
constexpr int ROW_WARPS = ROW_THREADS / 32;
constexpr int STAGES = 3;
constexpr int MAX_SEQS = 2048;
constexpr int PK = 128;            // keys per tile and query rows per item of the tensor-core prefix kernel
constexpr int PROWS = 256;

struct PoolView {
    const uint16_t* k;   // at the layer
    const uint16_t* v;
    long long k_page, k_head, v_page, v_head;   // elements
    int pages, page;
};

// What the join needs to know of a token: where its items start on the work
// line (kv head 0, row tile 0), how long one is, and the token's first row.
struct TokInfo {
    long long own_base, pfx_base;
    int own_ng, own_nrt, own_r0;
    int pfx_ng, pfx_nrt, pfx_r0, pfx_rows;
};

// Part rows are m, l, pad, pad, acc[D].  A run's split item sits in slot
// 2 * worker + 1 when the run has the item's start, else in slot 2 * worker;
// a whole item with another part beside it sits at its output row.
struct WsView {
    long long* head;    // [0] the call's arguments were in order, [1] groups per warp, [2] prefix tiles per CTA
    TokInfo* tok;       // [total_q]
    float* own_rowp;    // [total_q * Hq][D + 4]
    float* slots;       // [2 * warps][RT][D + 4]
    float* pfx_rowp;    // [total_q * Hq][D + 4], twice that with the tensor-core prefix (its two streams)
    float* pfx_slots;   // [2 * CTAs][PROWS][D + 4], tensor-core prefix only
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
    int B, NG, total_q, hq, hkv, top_k;
    int tc;                 // prefixes run on the tensor-core kernel
    float scale_log2;
    int* status;
    WsView ws;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a) : "memory");
}

// ---- the work line of an attend call --------------------------------------------------
// Entities: the groups' shared prefixes, then the sequences' own parts.  Built
// by every CTA for itself in shared memory (a few loads per sequence; a launch
// of its own would cost more).
struct Sched {
    long long* off;   // [NG + B + 1] groups of 16 positions before entity e, for one kv head
    int* len;         // [B] length of the sequence, 0 when its slot is wrong
    int* grp;         // [B] its group, or -1
    int* eff;         // [NG] shared pages read for the whole group
    int* gs;          // [NG + 1]
};
__host__ __device__ inline size_t sched_bytes(int B, int NG) {
    return ((size_t)(NG + B + 1) * 8 + (size_t)B * 8 + (size_t)(2 * NG + 1) * 4 + 15) & ~(size_t)15;
}
__device__ inline Sched sched_of(uint8_t* p, int B, int NG) {
    Sched s;
    s.off = (long long*)p;
    s.len = (int*)(s.off + NG + B + 1);
    s.grp = s.len + B;
    s.eff = s.grp + B;
    s.gs = s.eff + NG;
    return s;
}

__device__ __forceinline__ int q_start(const RowArgs& a, int b) { return a.q_starts ? a.q_starts[b] : b; }

__device__ __forceinline__ int own_groups(const RowArgs& a, const Sched& s, int b) {
    const int lo = s.grp[b] >= 0 ? s.eff[s.grp[b]] * a.pool.page : 0;
    return s.len[b] > lo ? ceil_div(s.len[b] - lo, GRP) : 0;
}

// Groups (or tiles) of a prefix item and its rows, in the units of the kernel that runs it.
__device__ __forceinline__ int pfx_groups(const RowArgs& a, int eff) {
    return a.tc ? ceil_div(eff * a.pool.page, PK) : eff * (a.pool.page / GRP);
}
__device__ __forceinline__ int pfx_tiles(const RowArgs& a, int toks, int grp) {
    const int rt = a.tc ? PROWS : RT;
    return (int)(((long long)toks * grp + rt - 1) / rt);
}

// Returns false (for every thread) when the starts are out of order.  PFX: the
// prefixes alone (s.len and s.grp are not used).
template <bool PFX>
__device__ inline bool build_sched(const RowArgs& a, const Sched& s, long long* scratch /* [blockDim / 32] */) {
    const int tid = threadIdx.x, nt = blockDim.x;
    bool bad = false;
    for (int g = tid; a.NG && g <= a.NG; g += nt) {   // without groups there are no arrays of them
        const int x = a.group_starts[g];
        if (x < 0 || x > a.B) bad = true;
        s.gs[g] = x;   // used only when every start is in order
        if (g < a.NG) {
            if (a.group_starts[g + 1] < x) bad = true;
            s.eff[g] = min(max(a.prefix_pages[g], 0), a.cols);
        }
    }
    if (a.q_starts) {
        for (int b = tid; b < a.B; b += nt)
            if (a.q_starts[b + 1] < a.q_starts[b]) bad = true;
        if (tid == 0 && (a.q_starts[0] != 0 || a.q_starts[a.B] != a.total_q)) bad = true;
    }
    if (__syncthreads_or(bad)) return false;
    for (int b = tid; b < a.B; b += nt) {
        const int slot = a.slots[b], ql = q_start(a, b + 1) - q_start(a, b);
        int len = 0;
        if (slot < 0 || slot >= a.num_slots) {
            if (!PFX && blockIdx.x == 0) note_status(a.status, MQ_ERR_BAD_SLOT);
        } else {
            len = a.lengths[slot];
            if (len < 0 || pages_of(len, a.pool.page) > a.cols) {
                if (!PFX && blockIdx.x == 0) note_status(a.status, MQ_ERR_BAD_POSITION);
                len = 0;
            }
        }
        int g = -1;
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
        // the shared part ends where the first query token of any member stands, so all its rows see all of it
        if (g >= 0 && ql > 0) atomicMin(&s.eff[g], max(0, len - ql) / a.pool.page);
    }
    __syncthreads();
    for (int g = tid; g < a.NG; g += nt)
        if (s.gs[g + 1] - s.gs[g] < 2) s.eff[g] = 0;   // a group of one shares nothing
    __syncthreads();
    const int E = a.NG + (PFX ? 0 : a.B), grp = a.hq / a.hkv;
    const int per = ceil_div(E, nt), e0 = min(E, tid * per), e1 = min(E, e0 + per);
    auto cost = [&](int e) -> long long {
        if (e < a.NG)
            return (long long)pfx_tiles(a, q_start(a, s.gs[e + 1]) - q_start(a, s.gs[e]), grp) * pfx_groups(a, s.eff[e]);
        const int b = e - a.NG;
        return ((q_start(a, b + 1) - q_start(a, b)) * (long long)grp + RT - 1) / RT * own_groups(a, s, b);
    };
    long long sum = 0;
    for (int e = e0; e < e1; ++e) sum += cost(e);
    const int lane = tid & 31, warp = tid >> 5;
    long long x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) scratch[warp] = x;
    __syncthreads();
    long long at = x - sum;
    for (int w = 0; w < warp; ++w) at += scratch[w];
    for (int e = e0; e < e1; ++e) {
        s.off[e] = at;
        at += cost(e);
    }
    if (tid == nt - 1) s.off[E] = at;
    __syncthreads();
    return true;
}

// Groups per warp: an equal share, but at least two, so that a short call is
// not cut into more parts than its join is worth.
__host__ __device__ __forceinline__ long long quota_of(long long work, long long warps) {
    const long long q = (work + warps - 1) / warps;
    return q < 2 ? 2 : q;
}

// One warp's 16-position group step and item bookkeeping.
template <typename T, int D>
struct RowWarp {
    static constexpr int TILE = GRP * D * 2;         // bytes of one K or V group
    static constexpr int STAGE = 2 * TILE;
    static constexpr int RING = STAGES * STAGE;
    static constexpr int CH = D / 8;                  // 16-byte chunks per row
    static constexpr int KS = D / 16;                 // k-steps of Q K^T
    static constexpr int LD = D + 4;                  // floats of a stored part row: m, l, pad, pad, acc

    uint32_t ring;     // this warp's ring, shared-memory address
    int lane;
    uint32_t qa[KS][4];
    float o[D / 8][4];
    float m[2], l[2];

    __device__ __forceinline__ void load_q(const RowArgs& a, int tok0, int h, int grp, int r0, int rows) {
        const int g = lane >> 2, t = lane & 3;
        const uint16_t* p[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + g + 8 * i;
            p[i] = g + 8 * i < rows ? a.q + (long long)(tok0 + r / grp) * a.q_tok + (h * grp + r % grp) * a.q_head : nullptr;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t* x = p[i & 1];
                qa[k][i] = x ? *reinterpret_cast<const uint32_t*>(x + 16 * k + 8 * (i >> 1) + 2 * t) : 0u;
            }
    }

    // Rows 0 .. vis - 1 of the group at row `row` of page `pid`, zeros past them.
    __device__ __forceinline__ void issue(const RowArgs& a, int stage, int pid, int row, int h, int vis) {
        const uint16_t* kp = a.pool.k + pid * a.pool.k_page + h * a.pool.k_head + row * D;
        const uint16_t* vp = a.pool.v + pid * a.pool.v_page + h * a.pool.v_head + row * D;
        const uint32_t s = ring + stage * STAGE;
#pragma unroll
        for (int j = 0; j < GRP * CH / 32; ++j) {
            const int c = lane + 32 * j, r = c / CH, x = c % CH;
            const uint32_t off = r * (D * 2) + ((x ^ (r & 7)) << 4);
            const bool ok = r < vis;
            cp16(s + off, ok ? kp + r * D + x * 8 : a.pool.k, ok);
            cp16(s + TILE + off, ok ? vp + r * D + x * 8 : a.pool.v, ok);
        }
    }

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    // lim0 / lim1: positions of the group (0 .. 16) that rows g and g + 8 see.
    // `mixed`: the rows of the tile do not all see the same positions.
    __device__ __forceinline__ void step(int stage, int lim0, int lim1, bool mixed, float scale) {
        const uint32_t ks = ring + stage * STAGE, vs = ks + TILE;
        const int t = lane & 3;
        const int mat = lane >> 3, r8 = lane & 7;
        float s[2][4], s2[2][4];   // two chains per tile: even and odd k-steps
#pragma unroll
        for (int i = 0; i < 4; ++i) s[0][i] = s[1][i] = s2[0][i] = s2[1][i] = 0.f;
        const int krow = (mat >> 1) * 8 + r8;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint32_t b0, b1, b2, b3;
            ldsm4(ks + krow * (D * 2) + (((2 * k + (mat & 1)) ^ r8) << 4), b0, b1, b2, b3);
            Elem<T>::mma(k & 1 ? s2[0] : s[0], qa[k], b0, b1);
            Elem<T>::mma(k & 1 ? s2[1] : s[1], qa[k], b2, b3);
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int p = 8 * n + 2 * t + (i & 1);
                const float x = (s[n][i] + s2[n][i]) * scale;
                s[n][i] = p < (i < 2 ? lim0 : lim1) ? x : -INFINITY;
                mx[i >> 1] = fmaxf(mx[i >> 1], s[n][i]);
            }
        float corr[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            const float mn = fmaxf(m[i], mx[i]);
            corr[i] = mn == m[i] ? 1.f : exp2f(m[i] - mn);   // m = -inf: nothing summed yet
            m[i] = mn;
        }
        const float u0 = m[0] == -INFINITY ? 0.f : m[0], u1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n][0] = exp2f(s[n][0] - u0);
            s[n][1] = exp2f(s[n][1] - u0);
            s[n][2] = exp2f(s[n][2] - u1);
            s[n][3] = exp2f(s[n][3] - u1);
        }
        l[0] = l[0] * corr[0] + ((s[0][0] + s[0][1]) + (s[1][0] + s[1][1]));
        l[1] = l[1] * corr[1] + ((s[0][2] + s[0][3]) + (s[1][2] + s[1][3]));
        if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                o[i][0] *= corr[0];
                o[i][1] *= corr[0];
                o[i][2] *= corr[1];
                o[i][3] *= corr[1];
            }
        }
        // P as the A operand, in two pieces of the 16-bit type (value and
        // remainder): one piece would cost as much accuracy as rounding the output does
        uint32_t pa[4], pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = s[i >> 1][2 * (i & 1)], y = s[i >> 1][2 * (i & 1) + 1];
            pa[i] = Elem<T>::pack(x, y);
            const float2 b = Elem<T>::up2(pa[i]);
            pr[i] = Elem<T>::pack(x - b.x, y - b.y);
        }
        const int vrow = (mat & 1) * 8 + r8;
        bool slow = false;
        if (mixed) {   // a masked weight of zero must not meet an infinity or NaN
            bool odd = false;
#pragma unroll
            for (int j = 0; j < GRP * CH / 32; ++j) {
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
        if (!slow) {
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                uint32_t b0, b1, b2, b3;
                ldsm4t(vs + vrow * (D * 2) + (((2 * n + (mat >> 1)) ^ r8) << 4), b0, b1, b2, b3);
                Elem<T>::mma(o[2 * n], pa, b0, b1);
                Elem<T>::mma(o[2 * n + 1], pa, b2, b3);
                Elem<T>::mma(o[2 * n], pr, b0, b1);
                Elem<T>::mma(o[2 * n + 1], pr, b2, b3);
            }
        } else {
            // one position at a time, added only to the rows that see it
#pragma unroll 1
            for (int p = 0; p < GRP; ++p) {
                uint32_t qa1[4], qr1[4], keep[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)   // this lane's columns 8 i + 2 t and + 1
                    keep[i] = p == 8 * i + 2 * t ? 0xffffu : p == 8 * i + 2 * t + 1 ? 0xffff0000u : 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    qa1[i] = pa[i] & keep[i >> 1];
                    qr1[i] = pr[i] & keep[i >> 1];
                }
#pragma unroll
                for (int n = 0; n < D / 16; ++n) {
                    uint32_t b[4];
                    ldsm4t(vs + vrow * (D * 2) + (((2 * n + (mat >> 1)) ^ r8) << 4), b[0], b[1], b[2], b[3]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x[4] = {0.f, 0.f, 0.f, 0.f};
                        Elem<T>::mma(x, qa1, b[2 * e] & keep[0], b[2 * e + 1] & keep[1]);
                        Elem<T>::mma(x, qr1, b[2 * e] & keep[0], b[2 * e + 1] & keep[1]);
                        if (p < lim0) {
                            o[2 * n + e][0] += x[0];
                            o[2 * n + e][1] += x[1];
                        }
                        if (p < lim1) {
                            o[2 * n + e][2] += x[2];
                            o[2 * n + e][3] += x[3];
                        }
                    }
                }
            }
        }
    }

    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
    }
    // Row g + 8 i of the tile, unnormalised, to a part row.
    __device__ __forceinline__ void put_part(float* dst, int i) {
        const int t = lane & 3;
        if (t == 0) *reinterpret_cast<float2*>(dst) = make_float2(m[i], l[i]);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(dst + 4 + 8 * n + 2 * t) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
    }
    __device__ __forceinline__ void put_out(uint16_t* dst, int i) {
        const int t = lane & 3;
        const float inv = l[i] != 0.f ? 1.f / l[i] : 0.f;   // a row that sees nothing is zero (NaN stays NaN)
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<uint32_t*>(dst + 8 * n + 2 * t) = Elem<T>::pack(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
    }
};

// MODE 0: attend (prefixes and own parts from the schedule).  MODE 1: sparse
// (token t's item reads the pages selected[t][h][..], top_k of them).
template <typename T, int D, int MODE>
__global__ void __launch_bounds__(ROW_THREADS) rows_kernel(const RowArgs a) {
    using W = RowWarp<T, D>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long scratch[ROW_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long wid = (long long)blockIdx.x * ROW_WARPS + warp, warps = (long long)gridDim.x * ROW_WARPS;
    const int grp = a.hq / a.hkv, page = a.pool.page;
    pdl_wait();
    pdl_trigger();
    Sched s;
    long long work, origin = 0;   // where this kernel's work starts on the line
    const int sp_ng = MODE == 1 ? a.top_k * (page / GRP) : 0, sp_nrt = ceil_div(grp, RT);
    if (MODE == 0) {
        s = sched_of(smem + ROW_WARPS * W::RING, a.B, a.NG);
        const bool ok = build_sched<false>(a, s, scratch);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            if (!ok) note_status(a.status, MQ_ERR_INVALID_ARGUMENT);
            a.ws.head[0] = ok;
        }
        if (!ok) return;
        origin = a.tc ? s.off[a.NG] * a.hkv : 0;
        work = s.off[a.NG + a.B] * a.hkv - origin;
        if (blockIdx.x == 0 && threadIdx.x == 0) a.ws.head[1] = quota_of(work, warps);
        // the join's view of the line, a share of the sequences per CTA
        for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
            const int q0 = q_start(a, b), q1 = q_start(a, b + 1), g = s.grp[b];
            TokInfo ti = {};
            ti.own_base = s.off[a.NG + b] * a.hkv - origin;
            ti.own_ng = own_groups(a, s, b);
            ti.own_nrt = (int)(((long long)(q1 - q0) * grp + RT - 1) / RT);
            int g0 = 0;
            if (g >= 0 && s.eff[g] > 0) {
                g0 = q_start(a, s.gs[g]);
                ti.pfx_base = s.off[g] * a.hkv;
                ti.pfx_ng = pfx_groups(a, s.eff[g]);
                ti.pfx_rows = (q_start(a, s.gs[g + 1]) - g0) * grp;
                ti.pfx_nrt = pfx_tiles(a, q_start(a, s.gs[g + 1]) - g0, grp);
            }
            for (int i = q0 + threadIdx.x; i < q1; i += ROW_THREADS) {
                ti.own_r0 = (i - q0) * grp;
                ti.pfx_r0 = (i - g0) * grp;
                a.ws.tok[i] = ti;
            }
        }
    } else {
        work = (long long)a.total_q * a.hkv * sp_nrt * sp_ng;
    }
    const long long quota = quota_of(work, warps);
    long long x = wid * quota;
    const long long xe = min(x + quota, work);

    W w;
    w.lane = lane;
    w.ring = smem_u32(smem) + warp * W::RING;
    const int g = lane >> 2;
    while (x < xe) {
        // the item at x: entity, kv head, row tile, and the groups of it that are this warp's
        int tok0, h, rt, rows_all, ng, gi, slot, len = 0, ql = 0, base = 0;
        bool prefix = false, other = false;
        if (MODE == 0) {
            const long long xh = (x + origin) / a.hkv;
            int lo = 0, hi = a.NG + a.B;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s.off[mid] <= xh) lo = mid;
                else hi = mid;
            }
            prefix = lo < a.NG;
            int b0, b1;
            if (prefix) {
                b0 = s.gs[lo];
                b1 = s.gs[lo + 1];
                ng = s.eff[lo] * (page / GRP);
            } else {
                b0 = lo - a.NG;
                b1 = b0 + 1;
                ng = own_groups(a, s, b0);
                len = s.len[b0];
                other = s.grp[b0] >= 0 && s.eff[s.grp[b0]] > 0;
                base = other ? s.eff[s.grp[b0]] * page : 0;
            }
            tok0 = q_start(a, b0);
            ql = q_start(a, b1) - tok0;
            // a prefix is read through a member's row of the table; a member without query tokens may have none
            int bs = b0;
            if (prefix)
                while (q_start(a, bs + 1) == q_start(a, bs)) ++bs;
            slot = a.slots[bs];
            rows_all = ql * grp;
            const long long rel = x + origin - s.off[lo] * a.hkv;
            const int nrt = ceil_div(rows_all, RT), it = (int)(rel / ng);
            gi = (int)(rel - (long long)it * ng);
            h = it / nrt;
            rt = it - h * nrt;
        } else {
            ng = sp_ng;
            const long long it = x / ng;
            gi = (int)(x - it * ng);
            rt = (int)(it % sp_nrt);
            const long long th = it / sp_nrt;
            h = (int)(th % a.hkv);
            tok0 = (int)(th / a.hkv);
            slot = a.slots[tok0];
            rows_all = grp;
            len = a.positions[tok0] + 1;
        }
        const int n = (int)min((long long)(ng - gi), xe - x);
        const int r0 = rt * RT, rows = min(RT, rows_all - r0);
        w.load_q(a, tok0, h, grp, r0, rows);
        w.reset();
        // the positions that the tile's rows see: [base, lim(row)), lim rising with the row
        const int first = len - ql + 1;
        auto lim = [&](int r) -> int {
            return MODE == 1 || prefix ? (prefix ? ng * GRP : len) : first + (r0 + min(r, rows - 1)) / grp;
        };
        const int lim_lo = lim(0), lim_hi = lim(rows - 1), lim_a = lim(g), lim_b = lim(g + 8);

        // lane i of `ids` knows page and position of the i-th group of a batch of 32
        int ids = -1, at = 0;
        auto look = [&](int k0) {
            const int k = k0 + lane;
            bool want = false;
            ids = -1;
            at = 0;
            if (k < n) {
                if (MODE == 0) {
                    at = base + (gi + k) * GRP;
                    ids = a.table[slot * a.table_row + at / page];
                    want = true;
                } else {
                    const int per = page / GRP, j = (gi + k) / per;
                    const int c = a.selected[((long long)tok0 * a.hkv + h) * a.top_k + j];
                    if (c >= 0) {   // listed: the slot and the column are in range
                        at = c * page + (gi + k - j * per) * GRP;
                        ids = a.table[slot * a.table_row + c];
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
        int ids_n = -1, at_n = 0;   // the batch before, while the ring straddles two
        look(0);
        auto fetch = [&](int k) {
            if (k < n) {
                if (k && (k & 31) == 0) {
                    ids_n = ids;
                    at_n = at;
                    look(k);
                }
                const int pid = __shfl_sync(0xffffffffu, ids, k & 31), p0 = __shfl_sync(0xffffffffu, at, k & 31);
                if (pid >= 0) w.issue(a, k % STAGES, pid, p0 & (page - 1), h, lim_hi - p0);
            }
            cp_commit();
        };
#pragma unroll
        for (int k = 0; k < STAGES - 1; ++k) fetch(k);
        for (int k = 0; k < n; ++k) {
            fetch(k + STAGES - 1);
            cp_wait<STAGES - 1>();
            __syncwarp();
            // group k may belong to the batch before the one that was looked up last
            const bool old = (k >> 5) < (min(k + STAGES - 1, n - 1) >> 5);
            const int pid = __shfl_sync(0xffffffffu, old ? ids_n : ids, k & 31);
            const int p0 = __shfl_sync(0xffffffffu, old ? at_n : at, k & 31);
            if (pid >= 0) w.step(k % STAGES, lim_a - p0, lim_b - p0, lim_lo < min(p0 + GRP, lim_hi), a.scale_log2);
            __syncwarp();
        }
        cp_wait<0>();
        w.finish();
        const bool whole = n == ng;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = g + 8 * i;
            if (r >= rows) continue;
            const int tok = tok0 + (r0 + r) / grp, head = h * grp + (r0 + r) % grp;
            const long long row = (long long)tok * a.hq + head;
            if (!whole)
                w.put_part(a.ws.slots + ((2 * wid + (gi == 0)) * RT + r) * W::LD, i);
            else if (prefix || other)
                w.put_part((prefix ? a.ws.pfx_rowp : a.ws.own_rowp) + row * W::LD, i);
            else
                w.put_out(a.out + row * D, i);
        }
        x += n;
    }
}

// ---- the join ----------------------------------------------------------------------------
// SPLIT warps share a row (few rows, many parts) or each warp has its own.
template <typename T, int D, int MODE, int SPLIT>
__global__ void __launch_bounds__(256) join_kernel(const RowArgs a, long long row_warps) {
    constexpr int LD = D + 4, V = D / 32;
    __shared__ float sm_m[8], sm_l[8], sm_o[8][D];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long rowi = SPLIT > 1 ? blockIdx.x : (long long)blockIdx.x * 8 + warp;
    if (rowi >= (long long)a.total_q * a.hq) return;
    const int sub = SPLIT > 1 ? warp : 0;
    const int tok = (int)(rowi / a.hq), head = (int)(rowi - (long long)tok * a.hq), grp = a.hq / a.hkv;
    const int h = head / grp;
    uint16_t* out = a.out + rowi * D;
    // the row's parts: np0 of the prefix (sub of them per run), then np1 of its own
    const float *src0 = nullptr, *src1 = nullptr;
    long long step0 = 0, step1 = 0;   // floats between parts
    int np0 = 0, np1 = 0, sub0 = 1;
    long long first0 = 0, first1 = 0, sub_step0 = 0;   // the first part of a split item is one slot further on
    if (MODE == 0) {
        if (!a.ws.head[0]) {   // refused: zeros
            for (int d = threadIdx.x & (SPLIT > 1 ? 255 : 31); d < D; d += SPLIT > 1 ? 256 : 32) out[d] = 0;
            return;
        }
    }
    const long long quota =
        MODE == 0 ? a.ws.head[1]
                  : quota_of((long long)a.total_q * a.hkv * ceil_div(grp, RT) * (a.top_k * (a.pool.page / GRP)), row_warps);
    {
        int ng, r;
        long long start;
        if (MODE == 0) {
            const TokInfo& ti = a.ws.tok[tok];
            ng = ti.own_ng;
            r = ti.own_r0 + head % grp;
            start = ti.own_base + ((long long)h * ti.own_nrt + r / RT) * ng;
            if (ti.pfx_ng) {
                const int R = a.tc ? PROWS : RT, pr = ti.pfx_r0 + head % grp, in = pr % R;
                const long long ps = ti.pfx_base + ((long long)h * ti.pfx_nrt + pr / R) * ti.pfx_ng;
                const long long pq = a.tc ? a.ws.head[2] : quota, w0 = ps / pq;
                const int runs = (int)((ps + ti.pfx_ng - 1) / pq - w0) + 1;
                if (a.tc && min(PROWS, ti.pfx_rows - (pr - in)) <= 128) sub0 = 2;   // both streams worked on this row
                np0 = runs * sub0;
                if (runs == 1) {
                    src0 = a.ws.pfx_rowp + rowi * LD;
                    sub_step0 = (long long)a.total_q * a.hq * LD;
                } else {
                    src0 = (a.tc ? a.ws.pfx_slots : a.ws.slots) + (2 * w0 * R + in) * LD;
                    step0 = 2ll * R * LD;
                    first0 = (long long)R * LD;
                    sub_step0 = 128ll * LD;
                }
            }
        } else {
            const int nrt = ceil_div(grp, RT);
            r = head % grp;
            ng = a.top_k * (a.pool.page / GRP);
            start = (((long long)tok * a.hkv + h) * nrt + r / RT) * ng;
        }
        if (ng) {
            const long long w0 = start / quota;
            np1 = (int)((start + ng - 1) / quota - w0) + 1;
            if (np1 == 1) {
                if (!np0) return;   // written by the only warp that had it
                src1 = a.ws.own_rowp + rowi * LD;
            } else {
                src1 = a.ws.slots + (2 * w0 * RT + r % RT) * LD;
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
    float M = -INFINITY;
    for (int i = sub + SPLIT * lane; i < np; i += SPLIT * 32) M = fmaxf(M, __ldcg(part(i)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float U = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 4
    for (int i = sub; i < np; i += SPLIT) {
        const float* p = part(i);
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p));
        const float e = exp2f(ml.x - U);
        L += ml.y * e;
        if (V == 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p + 4) + lane);
            acc[0] += v.x * e; acc[1] += v.y * e; acc[V - 2] += v.z * e; acc[V - 1] += v.w * e;
        } else {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(p + 4) + lane);
            acc[0] += v.x * e; acc[1] += v.y * e;
        }
    }
    if (SPLIT > 1) {
        if (lane == 0) {
            sm_m[warp] = M;
            sm_l[warp] = L;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sm_o[warp][lane * V + i] = acc[i];
        __syncthreads();
        if (warp) return;
        float MM = -INFINITY;
#pragma unroll
        for (int k = 0; k < SPLIT; ++k) MM = fmaxf(MM, sm_m[k]);
        const float UU = MM == -INFINITY ? 0.f : MM;
        L = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
        for (int k = 0; k < SPLIT; ++k) {
            const float e = exp2f(sm_m[k] - UU);
            L += sm_l[k] * e;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += sm_o[k][lane * V + i] * e;
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
