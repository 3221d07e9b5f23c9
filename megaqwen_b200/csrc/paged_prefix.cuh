// A group's shared prefix on the 5th-generation tensor cores: many query rows
// (the group's tokens x its q heads per kv head) against the same pages.
//
// Work: items of (group, kv head, 256 query rows) x 128-key tiles, laid end to
// end and cut into equal runs, one per CTA (one CTA per SM).  Every row sees
// every key of the prefix (the schedule ends it before the first query token),
// so there is no mask but the end of the last tile.
//
// A CTA runs two streams, A and B, each with its own Q tile (128 rows), its own
// S / P buffer and its own O accumulator in TMEM (4 x 128 columns):
//   more than 128 rows: A and B are the two halves of the rows, and each K and
//     V tile is used by both;
//   up to 128 rows: both take the same rows, A the even tiles of the run and B
//     the odd ones, and leave two parts.
// While one stream's softmax runs, the tensor core works for the other:
//   PV_A(j), S_A(j+1) | PV_B(j), S_B(j+1) | ...
// P overwrites S in place as two 16-bit pieces (value and remainder, 64 columns
// each), so the weights keep 16 bits and more; that makes 24 MMAs of 128 x 128
// x 16 per tile and stream (1536 cycles) against 16384 exponentials (1024
// cycles of the special-function units): the tensor core bounds the tile when
// there are many rows, HBM when there are few.
//
// Warps: 0 K producer, 1 MMA (and TMEM owner), 2 V producer, 3-6 softmax of A,
// 7-10 softmax of B (a thread per row; also load Q and store the parts).  K and
// V come page by page through a rank-5 tensor map, so the pool's strides are
// free; V is taken as it lies ([key][dim], the MMA's MN-major B operand).
// Every wait is bounded and ends in the status word.
#pragma once

#include <type_traits>

#include "mq_tc.cuh"
#include "paged_attn.cuh"

namespace mq {
namespace paged {

constexpr int PATOM = 128 * 128;         // bytes of 128 rows x 64 elements, 128-byte swizzle
constexpr int PFX_THREADS = 352;
constexpr int PFX_MAX_GROUPS = 256;
constexpr long long PFX_TIMEOUT = 4000000000ll;   // cycles, about two seconds

template <int D>
struct PfxSmem {
    static constexpr int TILE = (D / 64) * PATOM;
    static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE, BAR = 6 * TILE;
    static constexpr int SCHED = BAR + 256;
    static constexpr size_t bytes(int NG) { return SCHED + (size_t)(NG + 1) * 8 + (size_t)(2 * NG + 1) * 4 + 16 + 1024; }
};

struct PfxSeg {
    int g, h, r0, rows, t0, n, ng;   // rows: of this item (up to 256), r0: its first row in the group
    bool two;                        // both streams have rows of their own
    bool start, whole;
};

// MN-major operand in the 128-byte swizzle layout: 64 elements (128 B) per row
// of K, 8-row groups 1024 B apart, the next 64 elements `PATOM` away.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3fffu);
    d |= (uint64_t)(PATOM >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}

template <typename T>
__device__ constexpr uint32_t pfx_idesc(int N, bool b_mn) {
    const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;   // bf16 or f16, the same for A and B
    return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int x, int row, int h, int l, int p,
                                            uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(row), "r"(h), "r"(l), "r"(p), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Tiles per CTA: an equal share, at least two (both streams have one).
__host__ __device__ __forceinline__ long long pfx_quota(long long work, long long ctas) { return quota_of(work, ctas); }

template <typename T, int D>
__global__ void __launch_bounds__(PFX_THREADS, 1)
prefix_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const RowArgs a, int layer) {
    using L = PfxSmem<D>;
    constexpr int TILE = L::TILE, LD = D + 4;
    extern __shared__ uint8_t pfx_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pfx_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR);
    uint64_t* q_full = bars;          // [2] streams
    uint64_t* k_full = bars + 2;      // [2] stages
    uint64_t* k_empty = bars + 4;
    uint64_t* v_full = bars + 6;
    uint64_t* v_empty = bars + 8;
    uint64_t* s_full = bars + 10;     // [2] streams: S is there (and every MMA issued before it is done)
    uint64_t* p_full = bars + 12;     // [2] P is stored, O is rescaled
    uint64_t* o_full = bars + 14;     // [2] the run's last PV is done
    uint64_t* drain = bars + 16;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 17);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
    __shared__ long long scratch[PFX_THREADS / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 4);
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
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

    Sched s;
    s.off = reinterpret_cast<long long*>(smem + L::SCHED);
    s.eff = reinterpret_cast<int*>(s.off + a.NG + 1);
    s.gs = s.eff + a.NG;
    s.len = s.grp = nullptr;
    const bool in_order = build_sched<true>(a, s, scratch);
    const long long work = in_order ? s.off[a.NG] * a.hkv : 0;
    const long long quota = pfx_quota(work, gridDim.x);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.ws.head[2] = quota;
    const long long x0 = blockIdx.x * quota, xe = min(x0 + quota, work);
    const int grp = a.hq / a.hkv, page = a.pool.page;

    auto segment = [&](long long x) {
        PfxSeg e;
        const long long xh = x / a.hkv;
        int lo = 0, hi = a.NG;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s.off[mid] <= xh) lo = mid;
            else hi = mid;
        }
        e.g = lo;
        e.ng = ceil_div(s.eff[lo] * page, PK);
        const long long rel = x - s.off[lo] * a.hkv;
        const int all = (q_start(a, s.gs[lo + 1]) - q_start(a, s.gs[lo])) * grp;
        const int nrt = ceil_div(all, PROWS), it = (int)(rel / e.ng);
        e.t0 = (int)(rel - (long long)it * e.ng);
        e.h = it / nrt;
        e.r0 = (it - e.h * nrt) * PROWS;
        e.rows = min(PROWS, all - e.r0);
        e.two = e.rows > 128;
        e.n = (int)min((long long)(e.ng - e.t0), xe - x);
        e.start = e.t0 == 0;
        e.whole = e.n == e.ng;
        return e;
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        const long long t0 = clock64();
        while (!mbar_try_wait(bar, parity)) {
            if (*abort_flag || clock64() - t0 > PFX_TIMEOUT) return false;
        }
        return true;
    };
    auto give_up = [&]() {
        *abort_flag = 1;
        note_status(a.status, MQ_ERR_PIPE_TIMEOUT);
    };

    if (warp == 0 || warp == 2) {
        // ---- K and V producers: lane c loads the tile's c-th page (or half row block) ----
        uint64_t* full = warp == 0 ? k_full : v_full;
        uint64_t* empty = warp == 0 ? k_empty : v_empty;
        const CUtensorMap* map = warp == 0 ? &tmK : &tmV;
        uint8_t* ring = smem + (warp == 0 ? L::K : L::V);
        const int chunks = PK / page;
        int c = 0;   // tiles so far
        bool ok = true;
        for (long long x = x0; ok && x < xe;) {
            const PfxSeg e = segment(x);
            int b = s.gs[e.g];   // any member's row of the table will do; one without query tokens may have none
            while (q_start(a, b + 1) == q_start(a, b)) ++b;
            const int* row = a.table + a.slots[b] * a.table_row;
            const int last = s.eff[e.g] - 1;
            // past the end of the prefix the last page is loaded again: its scores are masked, and its
            // values (not stale shared memory) meet the zero weights
            auto look = [&](int j) { return lane < chunks ? row[min((e.t0 + j) * chunks + lane, last)] : 0; };
            int next = look(0);
            for (int j = 0; j < e.n; ++j, ++c) {
                int pid = next;
                if (j + 1 < e.n) next = look(j + 1);
                if (lane < chunks && (pid < 0 || pid >= a.pool.pages)) {
                    note_status(a.status, MQ_ERR_BAD_PAGE);
                    pid = a.pool.pages;   // outside the map: zeros
                }
                const int st = c & 1;
                bool here = c < 2 || wait(&empty[st], ((c >> 1) - 1) & 1);
                if (!__all_sync(0xffffffffu, here)) {
                    ok = false;
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(&full[st], TILE);
                __syncwarp();
                if (lane < chunks) {
#pragma unroll
                    for (int i = 0; i < D / 64; ++i)
                        tma_load_5d(ring + st * TILE + i * PATOM + lane * page * 128, map, 64 * i, 0, e.h, layer, pid, &full[st]);
                }
            }
            x += e.n;
        }
        if (!ok && lane == 0) give_up();
        // copies in flight land before the CTA may end, whatever became of their readers
        for (int k = max(0, c - 2); k < c; ++k) {
            const long long t0 = clock64();
            while (!mbar_try_wait(&full[k & 1], (k >> 1) & 1) && clock64() - t0 < PFX_TIMEOUT) {
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t id_s = pfx_idesc<T>(PK, false), id_o = pfx_idesc<T>(D, true);
            int c = 0;                          // K tiles of the segments before
            int np[2] = {0, 0};                 // PVs issued per stream
            int nq[2] = {0, 0};                 // Q tiles used per stream
            bool ok = true;
            for (long long x = x0; ok && x < xe;) {
                const PfxSeg e = segment(x);
                int pend[2] = {-1, -1};         // the tile whose PV is due
                bool first[2] = {true, true};
                const int c0 = c;
                auto pv = [&](int q) -> bool {
                    const int j = pend[q], vc = c0 + j;
                    if (!wait(&p_full[q], np[q] & 1)) return false;
                    if (!wait(&v_full[vc & 1], (vc >> 1) & 1)) return false;
                    tc_fence_after();
                    const uint32_t sv = smem_u32(smem + L::V + (vc & 1) * TILE);
                    const uint32_t p = tmem + q * 128, o = tmem + 256 + q * 128;
#pragma unroll
                    for (int half = 0; half < 2; ++half)   // the values, then the remainders
#pragma unroll
                        for (int k = 0; k < PK / 16; ++k)
                            tc_mma_f16_ts(o, p + half * 64 + k * 8, sw128_mnmajor_desc(sv + k * 2048), id_o,
                                          !first[q] || half || k);
                    first[q] = false;
                    ++np[q];
                    pend[q] = -1;
                    if (!e.two || q == 1) tc_commit(&v_empty[vc & 1]);
                    return true;
                };
                const int steps = e.two ? 2 * e.n : e.n;
                for (int i = 0; ok && i < steps; ++i) {
                    const int q = i & 1, j = e.two ? i >> 1 : i;
                    if (i < 2) {
                        ok = wait(&q_full[q], nq[q] & 1);
                        ++nq[q];
                        if (!ok) break;
                    }
                    if (pend[q] >= 0 && !pv(q)) {
                        ok = false;
                        break;
                    }
                    const int kc = c0 + j;
                    if (!wait(&k_full[kc & 1], (kc >> 1) & 1)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sq = smem_u32(smem + L::Q + q * TILE), sk = smem_u32(smem + L::K + (kc & 1) * TILE);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t off = (k >> 2) * PATOM + (k & 3) * 32;
                        tc_mma_f16(tmem + q * 128, sw128_kmajor_desc(sq + off), sw128_kmajor_desc(sk + off), id_s, k != 0);
                    }
                    tc_commit(&s_full[q]);
                    if (!e.two || q == 1) tc_commit(&k_empty[kc & 1]);
                    pend[q] = j;
                }
                // the last PV of each stream, the older tile first
                for (int i = 0; ok && i < 2; ++i) {
                    const int q = (steps + i) & 1;
                    if (pend[q] < 0) continue;
                    if (!pv(q)) {
                        ok = false;
                        break;
                    }
                    tc_commit(&o_full[q]);
                }
                c += e.n;
                x += e.n;
            }
            if (!ok) give_up();
            tc_commit(drain);   // MMAs in flight end before TMEM goes
            const long long t0 = clock64();
            while (!mbar_try_wait(drain, 0) && clock64() - t0 < PFX_TIMEOUT) {
            }
        }
    } else {
        // ---- softmax of stream q: a thread per row ----
        const int q = warp < 7 ? 0 : 1;
        const int quad = warp & 3;                     // the TMEM lanes this warp may touch
        const int r = quad * 32 + lane;
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const uint32_t sa = tmem + lane_off + q * 128, oa = tmem + lane_off + 256 + q * 128;
        constexpr float GROW = 8.f;
        int ns = 0, no = 0;
        bool ok = true;
        for (long long x = x0; ok && x < xe;) {
            const PfxSeg e = segment(x);
            x += e.n;
            const int mine = e.two ? e.n : (e.n + 1 - q) >> 1;   // this stream's tiles
            const int rr = e.two ? q * 128 + r : r;              // row in the item
            const bool live = rr < e.rows;
            const int row = e.r0 + rr, tok = q_start(a, s.gs[e.g]) + row / grp, head = e.h * grp + row % grp;
            const long long orow = (long long)tok * a.hq + head;
            float* part = nullptr;
            if (live)
                part = e.whole ? a.ws.pfx_rowp + ((e.two ? 0 : (long long)q * a.total_q * a.hq) + orow) * LD
                               : a.ws.pfx_slots + ((2ll * blockIdx.x + e.start) * PROWS + (e.two ? rr : q * 128 + r)) * LD;
            if (!mine) {   // a run of one tile: this stream's part is empty
                if (live)
                    for (int i = 0; i < LD; ++i) part[i] = i == 0 ? -INFINITY : 0.f;
                continue;
            }
            // Q rows, swizzled as TMA would; rows past the end are zero
            {
                uint8_t* dst = smem + L::Q + q * TILE + r * 128;
                const uint16_t* src = a.q + tok * a.q_tok + head * a.q_head;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const uint4 v = live ? *reinterpret_cast<const uint4*>(src + i * 8) : make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(dst + (i >> 3) * PATOM + (((i & 7) ^ (r & 7)) << 4)) = v;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[q]);
            }
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < mine; ++j, ++ns) {
                ok = wait(&s_full[q], ns & 1);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const int t = e.t0 + (e.two ? j : 2 * j + q);
                const int valid = s.eff[e.g] * page - t * PK;
                float sv[PK];
#pragma unroll
                for (int i = 0; i < PK; i += 32) tmem_ld32(sa + i, sv + i);
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < PK; ++i) sv[i] *= a.scale_log2;
                if (valid < PK) {
#pragma unroll
                    for (int i = 0; i < PK; ++i) sv[i] = i < valid ? sv[i] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < PK; ++i) mx[i & 3] = fmaxf(mx[i & 3], sv[i]);
                const float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
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
                        tmem_ld16(oa + i, v);
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[k] *= corr;
                        tmem_st16(oa + i, v);
                    }
                }
                const float u = m == -INFINITY ? 0.f : m;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < PK; i += 32) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float p0 = ex2(sv[i + 2 * k] - u), p1 = ex2(sv[i + 2 * k + 1] - u);
                        sum[k & 3] += p0 + p1;
                        hi[k] = Elem<T>::pack(p0, p1);
                        const float2 b = Elem<T>::up2(hi[k]);
                        lo[k] = Elem<T>::pack(p0 - b.x, p1 - b.y);
                    }
                    tmem_st16_nowait(sa + i / 2, hi);
                    tmem_st16_nowait(sa + 64 + i / 2, lo);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[q]);
            }
            if (!ok) break;
            ok = wait(&o_full[q], no & 1);
            ++no;
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            tc_fence_after();
            if (live) *reinterpret_cast<float4*>(part) = make_float4(m, l, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < D; i += 32) {
                float v[32];
                tmem_ld32(oa + i, v);
                if (live) {
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *reinterpret_cast<float4*>(part + 4 + i + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                }
            }
            tc_fence_before();
        }
        if (!ok && lane == 0) give_up();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace paged
}  // namespace mq
