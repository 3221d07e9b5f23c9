// A group's shared prefix on the 5th-generation tensor cores: many query rows
// (the group's tokens x its q heads per kv head) against the same pages.
//
// Work: items of (group, kv head, 256 query rows) x 128-key tiles, laid end to
// end and cut into equal runs, one per CTA (one CTA per SM).  Every row sees
// every key of the prefix (the schedule ends it before the first query token),
// so there is no mask but the end of the last tile (and pages that are out of range).
//
// A CTA runs two streams, A and B, each with its own Q tile (128 rows), its own
// S / P buffer and its own O accumulator in TMEM (4 x 128 columns):
//   more than 128 rows: A and B are the two halves of the rows, and each K and
//     V tile is used by both;
//   up to 128 rows: both take the same rows, A the even tiles of the run and B
//     the odd ones, and leave two parts.
// While one stream's softmax runs, the tensor core works for the other:
//   PV_A(j), S_A(j+1) | PV_B(j), S_B(j+1) | ...
// P overwrites S in place as two 16-bit pieces (value and remainder, side by
// side per 32 keys), so the weights keep 16 bits and more; that makes 24 MMAs of
// 128 x 128 x 16 per tile and stream, 1536 cycles, against 16384 exponentials,
// 1024 cycles of the special-function units.
//
// Bound: the chain softmax (2400 cycles) -> PV, S (1900 with commits) -> hand-over
// of a stream; the two streams overlap and a pair of tiles takes 5100 cycles.  32k
// keys x 256 rows x 8 kv heads: 57 us, 34 GFLOP without the remainders' MMAs (0.36
// of the measured bf16 rate; 51 GFLOP with them).  Few rows (8k x 128 x 8): 18 us
// for 34 MB, mostly a run's start and end (schedule 3.4 us, q and first tiles 5 us,
// parts 2.3 us).
//
// Warps: 0 K producer, 1 MMA (and TMEM owner), 2 V producer, 3-10 softmax of A,
// 11-18 softmax of B (two threads to a row, 64 keys each; they also load Q and
// store the parts; with one thread to a row 8k x 64 took 52 us and not 50).  K and
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
constexpr int PFX_THREADS = 608;
constexpr int PFX_MAX_GROUPS = 256;

template <int D>
struct PfxSmem {
    static constexpr int TILE = (D / 64) * PATOM;
    static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE, BAR = 6 * TILE;
    static constexpr int RED = BAR + 256;               // fp32 [2 streams][2 tiles][2 halves][128] row maxima
    static constexpr int SUM = RED + 2 * 2 * 2 * 128 * 4;   // fp32 [2 streams][2 halves][128] row sums
    static constexpr int SCHED = SUM + 2 * 2 * 128 * 4;
    static constexpr size_t bytes(int NG) { return SCHED + (size_t)(NG + 1) * 4 + (size_t)(2 * NG + 1) * 4 + 16 + 1024; }
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

// The same value in every lane, in a form the compiler knows to be uniform.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

template <typename P>
__device__ __forceinline__ P* from_lane(P* p, int lane) {
    return reinterpret_cast<P*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), lane));
}

__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r != 0;
}

// 64 consecutive 32-bit columns of this warp's TMEM lanes, waited for.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float* v) {
    uint32_t r[64];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

template <typename T, int D>
__global__ void __launch_bounds__(PFX_THREADS, 1)
prefix_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const RowArgs a) {
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
    __shared__ unsigned long long scratch[PFX_THREADS / 32];
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 8);
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 8);
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
    s.off = reinterpret_cast<uint32_t*>(smem + L::SCHED);
    s.eff = reinterpret_cast<int*>(s.off + a.NG + 1);
    s.gs = s.eff + a.NG;
    s.len = s.grp = nullptr;
    const bool in_order = build_sched<true, PFX_THREADS>(a, s, scratch);
    const uint32_t work = in_order ? s.off[a.NG] * a.hkv : 0;
    const uint32_t quota = quota_of(work, gridDim.x);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.ws.head[2] = quota;
    const uint32_t x0 = min(blockIdx.x * quota, work), xe = min(x0 + quota, work);
    const int grp = a.grp, page = a.pool.page;

    // The item at x and the tiles of it in this run (n <= 0: the run has only its own
    // units); x moves past them.
    auto segment = [&](uint32_t& x) {
        PfxSeg e;
        const uint32_t xh = x / (uint32_t)a.hkv;
        int lo = 0, hi = a.NG;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s.off[mid] <= xh) lo = mid;
            else hi = mid;
        }
        e.g = lo;
        e.ng = pfx_groups(a, s.eff[lo]);
        const uint32_t rel = x - s.off[lo] * a.hkv, len = e.ng + ITEM_UNITS, it = rel / len;
        const int pos = (int)(rel - it * len), left = (int)min(len - pos, xe - x);
        const int all = (q_start(a, s.gs[lo + 1]) - q_start(a, s.gs[lo])) * grp;
        const int nrt = pfx_tiles(a, all);
        e.t0 = max(pos - ITEM_UNITS, 0);
        e.n = max(pos + left - ITEM_UNITS, 0) - e.t0;
        e.h = (int)(it / (uint32_t)nrt);
        e.r0 = ((int)it - e.h * nrt) * PROWS;
        e.rows = min(PROWS, all - e.r0);
        e.two = e.rows > 128;
        e.start = e.t0 == 0;
        e.whole = e.n == e.ng;
        x += left;
        return e;
    };
    auto row_of = [&](const PfxSeg& e) -> const int* {
        int b = s.gs[e.g];   // any member's row of the table will do; one without query tokens may have none
        while (q_start(a, b + 1) == q_start(a, b)) ++b;
        return a.table + __ldg(a.slots + b) * a.table_row;
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

    if (warp == 0 || warp == 2) {
        // ---- K and V producers: lane c loads the tile's c-th page (or half row block) ----
        uint64_t* full = warp == 0 ? k_full : v_full;
        uint64_t* empty = warp == 0 ? k_empty : v_empty;
        const CUtensorMap* map = warp == 0 ? &tmK : &tmV;
        uint8_t* ring = smem + (warp == 0 ? L::K : L::V);
        const int chunks = PK / page;
        int c = 0;   // tiles so far
        bool ok = true;
        for (uint32_t x = x0; ok && x < xe;) {
            const PfxSeg e = segment(x);
            if (e.n <= 0) continue;
            const int* row = row_of(e);
            const int last = s.eff[e.g] - 1;
            // past the end of the prefix the last page is loaded again: its scores are masked, and its
            // values (not stale shared memory) meet the zero weights
            auto look = [&](int j) { return lane < chunks ? __ldg(row + min((e.t0 + j) * chunks + lane, last)) : 0; };
            int next = look(0);
            for (int j = 0; j < e.n; ++j, ++c) {
                int pid = next;
                if (j + 1 < e.n) next = look(j + 1);
                if (lane < chunks && (pid < 0 || pid >= a.pool.pages)) {
                    note_status(a.status, MQ_ERR_BAD_PAGE);
                    pid = a.pool.pages;   // outside the map: zeros (and its scores are masked)
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
                        tma_load_page(smem_u32(ring + st * TILE + i * PATOM + lane * page * 128), map, 0, i, e.h, pid, smem_u32(&full[st]));
                }
            }
        }
        if (!ok && lane == 0) give_up();
        // copies in flight land before the CTA may end, whatever became of their readers
        for (int k = max(0, c - 2); k < c; ++k) {
            const long long t0 = clock64();
            while (!mbar_try_wait(&full[k & 1], (k >> 1) & 1) && clock64() - t0 < WAIT_CYCLES) {
            }
        }
    } else if (warp == 1) {
        // ---- MMA: the whole warp walks, one elected lane issues.  All 512 columns of
        // TMEM are this CTA's, so their addresses start at 0 ----
        constexpr uint32_t id_s = pfx_idesc<T>(PK, false), id_o = pfx_idesc<T>(D, true);
        const uint32_t base = (smem_u32(pfx_raw) + 1023u) & ~1023u;
        int c0 = 0;                         // K tiles of the segments before
        uint32_t np0 = 0, np1 = 0;          // PVs issued per stream
        uint32_t nq0 = 0, nq1 = 0;          // Q tiles used per stream
        bool ok = true;
        auto scores = [&](int q, int kc, bool last_use) {
            const uint32_t sq = base + L::Q + q * TILE, sk = base + L::K + (kc & 1) * TILE;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint32_t off = (k >> 2) * PATOM + (k & 3) * 32;
                tc_mma_f16(q * 128, sw128_kmajor_desc(sq + off), sw128_kmajor_desc(sk + off), id_s, k != 0);
            }
            tc_commit(&s_full[q]);
            if (last_use) tc_commit(&k_empty[kc & 1]);
        };
        auto values = [&](int q, int vc, bool first, bool last_use, bool done) {
            const uint32_t sv = base + L::V + (vc & 1) * TILE, o = 256 + q * 128;
#pragma unroll
            for (int k = 0; k < PK / 16; ++k) {
                // 16 keys: 8 columns of values, the remainders 16 columns on
                const uint32_t p = q * 128 + 32 * (k >> 1) + 8 * (k & 1);
                const uint64_t dv = sw128_mnmajor_desc(sv + k * 2048);
                tc_mma_f16_ts(o, p, dv, id_o, !first || k);
                tc_mma_f16_ts(o, p + 16, dv, id_o, 1);
            }
            if (last_use) tc_commit(&v_empty[vc & 1]);
            if (done) tc_commit(&o_full[q]);
        };
        for (uint32_t x = x0; ok && x < xe;) {
            const PfxSeg e = segment(x);
            const int n = uniform(e.n);
            if (n <= 0) continue;
            const bool two = uniform(e.two);
            const int steps = two ? 2 * n : n;
            // step i: the stream's PV of its tile before (step i - 2), then its S of this one.  What the
            // step needs is waited for by four lanes at once.  (A second MMA warp, one for each stream, was
            // slower, 73 us against 58 for a 32k prefix: MMAs of two accumulators taking turns run slower than
            // runs of one.)
            for (int i = 0; ok && i < steps + 2; ++i) {
                const int q = i & 1;
                const bool pv = i >= 2, sc = i < steps;
                const int vc = c0 + (two ? (i - 2) >> 1 : i - 2), kc = c0 + (two ? i >> 1 : i);
                if (!pv && !sc) continue;   // a run of one tile: stream B has none
                uint64_t* bar = nullptr;
                uint32_t parity = 0;
                if (lane == 0 && sc) bar = &k_full[kc & 1], parity = kc >> 1;
                if (lane == 1 && pv) bar = &v_full[vc & 1], parity = vc >> 1;
                if (lane == 2 && pv) bar = &p_full[q], parity = q ? np1 : np0;
                if (lane == 3 && !pv) bar = &q_full[q], parity = q ? nq1 : nq0;
                ok = __all_sync(0xffffffffu, !bar || wait(bar, parity & 1));
                if (pv) (q ? np1 : np0)++;
                else (q ? nq1 : nq0)++;
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    if (pv) values(q, vc, i < 4, !two || q == 1, !sc);
                    if (sc) scores(q, kc, !two || q == 1);
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
        // ---- softmax of stream q, column half hh: a thread per row ----
        const int q = (warp - 3) >> 3, hh = ((warp - 3) >> 2) & 1;
        const int quad = warp & 3;                     // the TMEM lanes this warp may touch
        const int r = quad * 32 + lane;
        const float scale = fabsf(a.scale_log2);
        const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const uint32_t sa = tmem + lane_off + q * 128 + hh * 64, oa = tmem + lane_off + 256 + q * 128 + hh * (D / 2);
        float* red = reinterpret_cast<float*>(smem + L::RED) + q * 512;
        float* sums = reinterpret_cast<float*>(smem + L::SUM) + q * 256;
        constexpr float GROW = 8.f;
        // the two warps of a row meet at a barrier of their own; one whose wait failed goes on to the end
        // without waiting, so that its partner never stands alone
        auto meet = [&]() { named_bar_sync(1 + q * 4 + quad, 64); };
        int ns = 0, no = 0;
        bool ok = true;
        auto got = [&](uint64_t* bar, uint32_t parity) {
            if (ok) ok = __all_sync(0xffffffffu, wait(bar, parity));
            return ok;
        };
        for (uint32_t x = x0; x < xe;) {
            const PfxSeg e = segment(x);
            if (e.n <= 0) continue;
            const int mine = e.two ? e.n : (e.n + 1 - q) >> 1;   // this stream's tiles
            // lane k knows where row k of this warp comes from and where its part goes (a whole
            // item's to its output row, a split one's to a slot)
            const uint16_t* src = nullptr;
            float* part = nullptr;
            {
                const int wr = e.two ? q * 128 + r : r;
                if (wr < e.rows) {
                    const int t = (e.r0 + wr) / grp, head = e.h * grp + e.r0 + wr - t * grp, tok = q_start(a, s.gs[e.g]) + t;
                    src = a.q + tok * a.q_tok + head * a.q_head;
                    part = !e.whole ? a.ws.pfx_slots + ((2ll * blockIdx.x + e.start) * PROWS + q * 128 + r) * LD
                                    : a.ws.pfx_rowp + ((e.two ? 0 : (long long)q * a.total_q * a.hq) + (long long)tok * a.hq + head) * LD;
                }
            }
            if (!mine) {   // a run of one tile: this stream's part is empty (half the rows each, a row by all lanes)
#pragma unroll 1
                for (int k = hh * 16; k < hh * 16 + 16; ++k) {
                    float4* to = reinterpret_cast<float4*>(from_lane(part, k));
                    for (int i = lane; to && i < LD / 4; i += 32) to[i] = make_float4(i == 0 ? -INFINITY : 0.f, 0.f, 0.f, 0.f);
                }
                continue;
            }
            meet();   // both warps are done with the Q rows of the item before
            // Q rows, swizzled as TMA would, zeros past the end; a negative scale turns their
            // signs.  Half the rows each, LPR lanes side by side on a row, all loads in flight.
            {
                constexpr int LPR = D / 8, RPI = 32 / LPR, N = 16 / RPI;
                const int ch = lane % LPR, sub = lane / LPR;
                uint4 v[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint16_t* row = from_lane(src, hh * 16 + i * RPI + sub);
                    v[i] = row ? __ldg(reinterpret_cast<const uint4*>(row + ch * 8)) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int w = quad * 32 + hh * 16 + i * RPI + sub;
                    v[i].x ^= sign; v[i].y ^= sign; v[i].z ^= sign; v[i].w ^= sign;
                    *reinterpret_cast<uint4*>(smem + L::Q + q * TILE + (ch >> 3) * PATOM + w * 128 +
                                              (((ch & 7) ^ (w & 7)) << 4)) = v[i];
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[q]);
            }
            float m = -INFINITY, l = 0.f;
            // lane i: whether page `at + i` of the prefix is out of range (the last one, past the end)
            auto gone = [&](int at) {
                const int pid = __ldg(row_of(e) + min(at + lane, s.eff[e.g] - 1));
                return pid < 0 || pid >= a.pool.pages;
            };
            // looked up once per run, while the first scores are on their way, and again tile by tile only if there are any
            bool holes = false;
#pragma unroll 1
            for (int i = 0; i < e.n * (PK / page); i += 32) holes |= gone(e.t0 * (PK / page) + i);
            holes = __any_sync(0xffffffffu, holes);
            for (int j = 0; j < mine; ++j, ++ns) {
                float tmax = -INFINITY;
                const int t = e.t0 + (e.two ? j : 2 * j + q);
                const unsigned none = holes ? __ballot_sync(0xffffffffu, gone(t * (PK / page))) : 0u;
                if (got(&s_full[q], ns & 1)) {
                    tc_fence_after();
                    const int valid = s.eff[e.g] * page - t * PK - hh * 64;
                    // the end of the prefix, and pages that are not there: their scores are set to minus infinity in TMEM
                    if (valid < 64 || none) {
#pragma unroll 1
                        for (int i = 0; i < 64; i += 32) {
                            uint32_t live = valid >= i + 32 ? 0xffffffffu : valid > i ? (1u << (valid - i)) - 1u : 0u;
                            for (int k = 0; k < 32; k += 16)   // a page is 16 keys or more
                                if (none >> ((hh * 64 + i + k) >> a.pool.shift) & 1u) live &= ~(0xffffu << k);
                            float sv[32];
                            tmem_ld32(sa + i, sv);
#pragma unroll
                            for (int k = 0; k < 32; ++k) sv[k] = live >> k & 1u ? sv[k] : -INFINITY;
                            tmem_st32(sa + i, sv);
                        }
                    }
                    // two passes over S in TMEM: the code stays small (a run is a few tiles long, and
                    // fetching unrolled code the first time cost more than reading S twice)
                    float sv[64], mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    tmem_ld64(sa, sv);
#pragma unroll
                    for (int k = 0; k < 64; ++k) mx[k & 3] = fmaxf(mx[k & 3], sv[k]);
                    tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
                }
                red[((j & 1) * 2 + hh) * 128 + r] = tmax;
                meet();
                if (!ok) continue;
                tmax = fmaxf(tmax, red[((j & 1) * 2 + (hh ^ 1)) * 128 + r]);
                // a row's maximum moves only when it grew by more than 2^8; weights stay below 256
                float corr = 1.f;
                if (tmax > m + GROW) {
                    corr = ex2(m - tmax);   // 0 on the first tile
                    m = tmax;
                }
                l *= corr;
                if (j && __any_sync(0xffffffffu, corr != 1.f)) {
                    // s_full covers the PV before it, so O is at rest; half its columns each
#pragma unroll 1
                    for (int i = 0; i < D / 2; i += 16) {
                        float v[16];
                        tmem_ld16(oa + i, v);
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[k] *= corr;
                        tmem_st16(oa + i, v);
                    }
                }
                const float u = m == -INFINITY ? 0.f : m;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                for (int i = 0; i < 64; i += 32) {
                    float sv[32];
                    uint32_t pk[32];   // 32 weights in 16 columns, their remainders in the next 16
                    tmem_ld32(sa + i, sv);
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float p0 = ex2(fmaf(sv[2 * k], scale, -u)), p1 = ex2(fmaf(sv[2 * k + 1], scale, -u));
                        sum[k & 3] += p0 + p1;
                        pk[k] = Elem<T>::pack(p0, p1);
                        const float2 b = Elem<T>::up2(pk[k]);
                        pk[16 + k] = Elem<T>::pack(p0 - b.x, p1 - b.y);
                    }
                    tmem_st16_nowait(sa + i, pk);
                    tmem_st16_nowait(sa + i + 16, pk + 16);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[q]);
            }
            const bool done = got(&o_full[q], no & 1);
            ++no;
            sums[hh * 128 + r] = l;
            meet();
            if (!done) continue;
            tc_fence_after();
            l += sums[(hh ^ 1) * 128 + r];
            // the part rows, this half's columns, a quarter of D at a time through half of the row's bytes of
            // the Q tile (every S that reads it is done), so that lanes side by side write 64 or 128 bytes of a row
            if (part && hh == 0) *reinterpret_cast<float4*>(part) = make_float4(m, l, 0.f, 0.f);
            constexpr int W = D / 4, LPR = W / 4, RPI = 32 / LPR;
            auto stage = [&](int row, int c) -> float4* {   // 16-byte piece c of this half's share of a row
                const int at = D == 128 ? c : hh * 4 + c;
                return reinterpret_cast<float4*>(smem + L::Q + q * TILE + (D == 128 ? hh * PATOM : 0) + (quad * 32 + row) * 128 +
                                                 ((at ^ (row & 7)) << 4));
            };
#pragma unroll 1
            for (int i = 0; i < D / 2; i += W) {
                float v[W];
                if (W == 32) tmem_ld32(oa + i, v);
                else tmem_ld16(oa + i, v);
#pragma unroll
                for (int k = 0; k < W; k += 4) *stage(lane, k >> 2) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                __syncwarp();
                const int ch = lane % LPR, sub = lane / LPR;
#pragma unroll 4
                for (int k = sub; k < 32; k += RPI) {
                    float* to = from_lane(part, k);
                    if (to) *reinterpret_cast<float4*>(to + 4 + hh * (D / 2) + i + ch * 4) = *stage(k, ch);
                }
                __syncwarp();
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
