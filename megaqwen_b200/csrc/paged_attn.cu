// Attention over the paged cache: batches that share a prefix, and sparse
// attention over pages chosen by score.  Kernels in paged_attn.cuh; here the
// choice of pages and the host side.
#include <algorithm>
#include <type_traits>

#include "paged_attn.cuh"
#include "paged_by_page.cuh"
#include "paged_prefix.cuh"

namespace mq {

bool make_tmap_nd(CUtensorMap* map, const void* ptr, bool bf16, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                  const cuuint32_t* box);

namespace paged {

// ---- choosing pages -----------------------------------------------------------------------
// Scores of all earlier pages into shared memory as order-preserving 32-bit
// keys, then a radix selection of the (top_k - 1)-th largest over the bits in
// which the keys differ (8 at a time; a bin of up to 32 keys is ranked pair by
// pair), then the list in ascending order.  Reads 2 D + 1 bytes per page.  The
// products run on mma.sync m16n8k32 (16 pages, 8 columns, 32 channels; dp4a took
// 110 instructions for what is 8 MMAs with two heads): whole numbers, exact below
// 2^24, so the keys do not depend on their order.
//
// Two forms.  select_one_kernel: an item is a (kv head, token), a cluster of up to
// 8 CTAs to an item, each scoring a share of the pages; for few items, whose reads
// have to be spread.  select_eight_kernel: eight tokens of one kv head to a CTA,
// each page's record read once for all of them that stand in the same sequence;
// for many items (500 tokens x 8 heads, 250 pages each: 29 us; 54 with a warp to
// an item of its own, 121 with a CTA).
constexpr int MAX_SPARSE_COLS = 49152;
constexpr int MAX_SPARSE_GROUP = 64;   // q heads per kv head
constexpr int SEL_UNROLL = 2;          // of select_one_kernel: 16-page steps in flight
constexpr int SEL_WARPS = 16;          // of select_one_kernel
constexpr int SEL_TOKENS = 8;          // of select_eight_kernel, a warp each

struct SelArgs {
    const signed char* index;   // at the layer
    long long i_page, i_head;
    const uint16_t* q;
    long long q_tok, q_head;
    const int* table;
    long long table_row;
    const int* slots;
    const int* positions;
    int* selected;
    int n, num_slots, cols, pages, shift, hkv, grp, top_k;
    int* status;
    uint32_t* count;   // page by page: how many tokens chose (kv head, page), and each token's rank there
    int* rank;
};

__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float two_to(int e) { return __int_as_float((e + 127) << 23); }

// heads are padded to a multiple of 8 with zeros
template <int D>
size_t sel_one_bytes(int cols, int grp) {
    return (size_t)cols * 4 + (size_t)((grp + 7) & ~7) * (2 * D + 4);
}
template <int D>
size_t sel_eight_bytes(int cols, int grp) {
    return SEL_TOKENS * ((size_t)cols * 4 + (size_t)grp * (2 * D + 4));
}

__device__ __forceinline__ void mma_s8(int* d, const int* a, int b0, int b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One head of a query in whole numbers, split by sign, by one warp; returns the unit.
template <typename T, int D>
__device__ __forceinline__ float whole_query(const float (&x)[D / 32], signed char* pos, signed char* neg, int lane) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) m = fmaxf(m, fabsf(x[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = fminf(m, Elem<T>::MAX);
    const int e = m > 0.f ? min(max(ilogbf(m) - 6, -60), 40) : 0;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const float r = fminf(fmaxf(rintf(x[i] * two_to(-e)), -127.f), 127.f);
        const int v = x[i] == x[i] ? (int)r : 0;
        pos[lane + 32 * i] = (signed char)max(v, 0);
        neg[lane + 32 * i] = (signed char)min(v, 0);
    }
    return two_to(e);
}
template <typename T, int D>
__device__ __forceinline__ void load_query(float (&x)[D / 32], const uint16_t* q, int lane) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) x[i] = q ? Elem<T>::up(__ldg(q + lane + 32 * i)) : 0.f;
}

// 16 pages a step: lane (g, t) reads channels 16 t .. of each 64-channel block of
// pages g and g + 8, whose words are the A operand of two MMAs; the k index is
// permuted alike in both operands.  Blocks: HI, then LO.
template <int D>
struct PageStep {
    int4 w[2][2 * D / 64];
    int ex[2];
    __device__ __forceinline__ void load(const signed char* ix, long long i_page, const int (&pid)[2], int tq) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const signed char* rec = ix + (pid[r] >= 0 ? pid[r] : 0) * i_page;
#pragma unroll
            for (int b = 0; b < 2 * D / 64; ++b) w[r][b] = __ldg(reinterpret_cast<const int4*>(rec + 64 * b + 16 * tq));
            ex[r] = __ldg(rec + 2 * D);
        }
    }
    __device__ __forceinline__ void dot(int (&c)[4], const int4 (&q)[2 * D / 64]) const {
        c[0] = c[1] = c[2] = c[3] = 0;
#pragma unroll
        for (int b = 0; b < 2 * D / 64; ++b) {
            const int4 x = w[0][b], y = w[1][b];
            const int a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
            mma_s8(c, a0, q[b].x, q[b].y);
            mma_s8(c, a1, q[b].z, q[b].w);
        }
    }
    // the record's exponent is within [-60, 40] when this library wrote it
    __device__ __forceinline__ uint32_t key(int r, float score, bool there) const {
        return there ? order_key(score * two_to(min(max(ex[r], -60), 40))) : 0u;
    }
};

// What a selection needs beside its keys.
struct Picker {
    int* hist;        // [256]
    int* list;        // [32]
    uint32_t* pick;   // [4]
    int* ends;        // [2][NW] each warp's smallest and largest key
    int* sums;        // [2][NW] each warp's counts
};

// The `want` largest of keys[0 .. own - 1] (ties: the lowest first), 0 < want < own,
// as places in ascending order into sel.  NW warps together.
template <int NW>
__device__ __forceinline__ void choose(const uint32_t* keys, int own, int want, int* sel, const Picker& s, int warp, int lane) {
    constexpr int NT = NW * 32;
    const int tid = warp * 32 + lane;
    auto sync = [&]() {
        if (NW == 1) __syncwarp();
        else __syncthreads();
    };
    uint32_t kmin = 0xffffffffu, kmax = 0;
    for (int j = tid; j < own; j += NT) {
        kmin = min(kmin, keys[j]);
        kmax = max(kmax, keys[j]);
    }
    kmin = __reduce_min_sync(0xffffffffu, kmin);
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (NW > 1) {
        if (lane == 0) {
            s.ends[warp] = (int)kmin;
            s.ends[NW + warp] = (int)kmax;
        }
        __syncthreads();
        kmin = __reduce_min_sync(0xffffffffu, (uint32_t)s.ends[lane % NW]);
        kmax = __reduce_max_sync(0xffffffffu, (uint32_t)s.ends[NW + lane % NW]);
    }
    // keys agree above bit `bits`; of those that match `prefix` under `mask` the largest `need` are wanted
    int bits = 32 - __clz((int)(kmin ^ kmax)), need = want;
    uint32_t mask = bits == 32 ? 0u : 0xffffffffu << bits, prefix = kmax & mask;
    while (bits > 0) {
        const int shift = max(bits - 8, 0);
        for (int i = tid; i < 256; i += NT) s.hist[i] = 0;
        if (tid == 0) s.pick[2] = 0;
        sync();
        for (int j = tid; j < own; j += NT) {
            const uint32_t k = keys[j];
            if ((k & mask) == prefix) atomicAdd(&s.hist[(k & ~mask) >> shift], 1);
        }
        sync();
        if (warp == 0) {
            // lane i holds bins 255 - 8 i .. 248 - 8 i; the bin in which the count passes `need`
            int c[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                c[i] = s.hist[255 - 8 * lane - i];
                sum += c[i];
            }
            int x = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            int above = x - sum;
            if (above < need && need <= x) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (above < need && need <= above + c[i]) {
                        s.pick[0] = prefix | (uint32_t)(255 - 8 * lane - i) << shift;
                        s.pick[1] = (uint32_t)(need - above);   // wanted of the bin
                        s.pick[3] = (uint32_t)c[i];
                        above = need;   // found
                    } else {
                        above += c[i];
                    }
                }
            }
        }
        sync();
        prefix = s.pick[0];
        need = (int)s.pick[1];
        const int in_bin = (int)s.pick[3];
        mask = 0xffffffffu << shift;
        bits = shift;
        if (need == in_bin || bits == 0) break;   // all of the bin, or all its keys are equal
        if (in_bin <= 32) {
            // few keys: rank them against each other, equal ones by their place
            for (int j = tid; j < own; j += NT)
                if ((keys[j] & mask) == prefix) s.list[atomicAdd(&s.pick[2], 1u)] = j;
            sync();
            if (warp == 0) {
                const int at = lane < in_bin ? s.list[lane] : 0x7fffffff;
                const uint32_t k = lane < in_bin ? keys[at] : 0u;
                int rank = 0;
                for (int i = 0; i < in_bin; ++i) {
                    const uint32_t ki = __shfl_sync(0xffffffffu, k, i);
                    const int ai = __shfl_sync(0xffffffffu, at, i);
                    rank += ki > k || (ki == k && ai < at);
                }
                const unsigned last = __ballot_sync(0xffffffffu, lane < in_bin && rank == need - 1);
                const uint32_t low = __shfl_sync(0xffffffffu, k, __ffs((int)last) - 1);
                const unsigned same = __ballot_sync(0xffffffffu, lane < in_bin && rank < need && k == low);
                if (lane == 0) {
                    s.pick[0] = low;
                    s.pick[1] = (uint32_t)__popc(same);
                }
            }
            sync();
            prefix = s.pick[0];
            need = (int)s.pick[1];
            mask = 0xffffffffu;
            break;
        }
        sync();   // the pick is read before the next pass writes it
    }
    // keys above the bin, and the first `need` in it, in ascending order of the page
    const int seg = (ceil_div(own, NW) + 31) & ~31;
    const int lo = min(own, warp * seg), hi = min(own, lo + seg);
    int gt = 0, eq = 0;
    if (NW > 1) {
        for (int i = lo; i < hi; i += 32) {
            const uint32_t k = i + lane < hi ? keys[i + lane] & mask : 0u;
            gt += __popc(__ballot_sync(0xffffffffu, i + lane < hi && k > prefix));
            eq += __popc(__ballot_sync(0xffffffffu, i + lane < hi && k == prefix));
        }
        if (lane == 0) {   // (not into `ends`: with all keys equal no barrier lies between its reads and this)
            s.sums[warp] = gt;
            s.sums[NW + warp] = eq;
        }
        __syncthreads();
        gt = eq = 0;
        for (int w = 0; w < warp; ++w) {
            gt += s.sums[w];
            eq += s.sums[NW + w];
        }
    }
    const unsigned below = (1u << lane) - 1u;
    for (int i = lo; i < hi; i += 32) {
        const uint32_t k = i + lane < hi ? keys[i + lane] & mask : 0u;
        const bool is_gt = i + lane < hi && k > prefix, is_eq = i + lane < hi && k == prefix;
        const unsigned mg = __ballot_sync(0xffffffffu, is_gt), me = __ballot_sync(0xffffffffu, is_eq);
        const int eq_at = eq + __popc(me & below);
        if (is_gt || (is_eq && eq_at < need)) sel[gt + __popc(mg & below) + min(eq_at, need)] = i + lane;
        gt += __popc(mg);
        eq += __popc(me);
    }
}

// Where token t's choice is clear without scores (a wrong place, every page, only
// its own), writes it and returns 0; otherwise the number of pages to score.
// `write`: this group of nt threads writes.
__device__ __forceinline__ int pages_to_score(const SelArgs& a, int slot, int pos, int* sel, bool write, int tid, int nt) {
    const bool bad_slot = slot < 0 || slot >= a.num_slots;
    const int own = pos >> a.shift, want = a.top_k - 1;
    if (bad_slot || pos < 0 || own >= a.cols) {
        if (write && tid == 0) note_status(a.status, bad_slot ? MQ_ERR_BAD_SLOT : MQ_ERR_BAD_POSITION);
        for (int i = tid; write && i < a.top_k; i += nt) sel[i] = -1;
        return 0;
    }
    if (own <= want || want == 0) {
        for (int i = tid; write && i < a.top_k; i += nt) sel[i] = want == 0 ? own : i <= own ? i : -1;
        return 0;
    }
    return own;
}

template <typename T, int D>
__global__ void __launch_bounds__(SEL_WARPS * 32) select_one_kernel(const SelArgs a) {
    constexpr int NW = SEL_WARPS, NT = NW * 32;
    extern __shared__ __align__(16) uint8_t sel_smem[];
    __shared__ int hist[256], ends[2 * NW], sums[2 * NW], list[32];
    __shared__ uint32_t pick[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x;
    const int heads = (a.grp + 7) & ~7;
    signed char* qpos = reinterpret_cast<signed char*>(sel_smem);          // [heads][D]
    signed char* qneg = qpos + heads * D;
    float* qunit = reinterpret_cast<float*>(qneg + heads * D);             // [heads]
    uint32_t* keys = reinterpret_cast<uint32_t*>(qunit + heads);           // [cols]
    pdl_wait();
    pdl_trigger();
    const uint32_t rank = cluster_rank(), ranks = cluster_size();
    const uint32_t item = blockIdx.x / ranks;
    const int h = (int)(item / (uint32_t)a.n), t = (int)(item - (uint32_t)h * a.n);
    int* sel = a.selected + ((long long)t * a.hkv + h) * a.top_k;
    const int slot = __ldg(a.slots + t);
    const int own = pages_to_score(a, slot, __ldg(a.positions + t), sel, rank == 0, tid, NT);
    if (!own) return;   // all CTAs of the cluster alike
    // this CTA's share of the pages, looked up in one sweep; each place is overwritten by its page's key
    const int share = ranks == 1 ? own : (ceil_div(own, (int)ranks) + 15) & ~15;
    const int p0 = min(own, (int)rank * share), p1 = min(own, p0 + share);
    const int* row = a.table + slot * a.table_row;
    const uint16_t* q0 = a.q + t * a.q_tok + (long long)h * a.grp * a.q_head;
    float x[D / 32];   // a warp's first head is on its way before the sweep
    load_query<T, D>(x, warp < a.grp ? q0 + warp * a.q_head : nullptr, lane);
    for (int j0 = p0; j0 < p1; j0 += 4 * NT) {
        int pid[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pid[i] = j0 + i * NT + tid < p1 ? __ldg(row + j0 + i * NT + tid) : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + i * NT + tid;
            if (j >= p1) break;
            if (pid[i] < 0 || pid[i] >= a.pages) {
                note_status(a.status, MQ_ERR_BAD_PAGE);
                pid[i] = -1;
            }
            keys[j] = (uint32_t)pid[i];
        }
    }
    for (int g = warp; g < heads; g += NW) {
        if (g != warp) load_query<T, D>(x, g < a.grp ? q0 + g * a.q_head : nullptr, lane);
        const float unit = whole_query<T, D>(x, qpos + g * D, qneg + g * D, lane);
        if (lane == 0) qunit[g] = unit;
    }
    if (ranks > 1) cluster_sync();   // (every CTA runs: its shared memory may be written)
    else __syncthreads();
    const int g = lane >> 2, tq = lane & 3;
    const signed char* ix = a.index + h * a.i_head;
#pragma unroll 1
    for (int j0 = p0 + warp * 16; j0 < p1; j0 += NW * 16 * SEL_UNROLL) {
        PageStep<D> st[SEL_UNROLL];
        int pid[SEL_UNROLL][2];
#pragma unroll
        for (int u = 0; u < SEL_UNROLL; ++u) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int j = j0 + u * NW * 16 + g + 8 * r;
                pid[u][r] = j < p1 ? (int)keys[j] : -1;
            }
            st[u].load(ix, a.i_page, pid[u], tq);
        }
        float best[SEL_UNROLL][2];
#pragma unroll
        for (int u = 0; u < SEL_UNROLL; ++u) best[u][0] = best[u][1] = -INFINITY;
        for (int h0 = 0; h0 < a.grp; h0 += 8) {   // columns: 8 heads
            int4 q[2 * D / 64];
#pragma unroll
            for (int b = 0; b < 2 * D / 64; ++b)
                q[b] = *reinterpret_cast<const int4*>((b < D / 64 ? qpos : qneg) + (h0 + g) * D + (b % (D / 64)) * 64 + 16 * tq);
            const float u0 = qunit[h0 + 2 * tq], u1 = qunit[h0 + 2 * tq + 1];
            const bool in0 = h0 + 2 * tq < a.grp, in1 = h0 + 2 * tq + 1 < a.grp;
#pragma unroll
            for (int u = 0; u < SEL_UNROLL; ++u) {
                int c[4];
                st[u].dot(c, q);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    if (in0) best[u][r] = fmaxf(best[u][r], (float)c[2 * r] * u0);
                    if (in1) best[u][r] = fmaxf(best[u][r], (float)c[2 * r + 1] * u1);
                }
            }
        }
        __syncwarp();   // the page numbers are read
#pragma unroll
        for (int u = 0; u < SEL_UNROLL; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float s = best[u][r];
                s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, 1));
                s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, 2));
                const int j = j0 + u * NW * 16 + g + 8 * r;
                if (j < p1 && tq == 0) {
                    const uint32_t key = st[u].key(r, s, pid[u][r] >= 0);
                    if (rank == 0) keys[j] = key;
                    else st_peer(smem_u32(keys + j), 0, key);   // places that the first CTA uses for nothing else
                }
            }
    }
    if (ranks > 1) {
        cluster_sync();   // every share is scored and in the first CTA
        if (rank) return;
    } else {
        __syncthreads();
    }
    choose<NW>(keys, own, a.top_k - 1, sel, {hist, list, pick, ends, sums}, warp, lane);
    if (tid == 0) sel[a.top_k - 1] = own;
}

template <typename T, int D>
__global__ void __launch_bounds__(SEL_TOKENS * 32, 3) select_eight_kernel(const SelArgs a) {
    // one 16-page step in flight, three CTAs to an SM: 29 us for 500 tokens; two steps, two CTAs: 32
    constexpr int N = SEL_TOKENS, UNROLL = 1;
    extern __shared__ __align__(16) uint8_t sel_smem[];
    __shared__ int hist[N][256], list[N][32], owns[N], slot_of[N];
    __shared__ uint32_t pick[N][4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    signed char* qpos = reinterpret_cast<signed char*>(sel_smem);          // [grp][N][D]
    signed char* qneg = qpos + a.grp * N * D;
    float* qunit = reinterpret_cast<float*>(qneg + a.grp * N * D);         // [grp][N]
    uint32_t* keys = reinterpret_cast<uint32_t*>(qunit + a.grp * N);       // [N][cols]
    pdl_wait();
    pdl_trigger();
    const int blocks = ceil_div(a.n, N), h = blockIdx.x / blocks, t = (blockIdx.x - h * blocks) * N + warp;
    // a warp to a token: what it has to choose from, its queries
    int own = 0, slot = -1;
    int* sel = a.selected + ((long long)t * a.hkv + h) * a.top_k;
    if (t < a.n) {
        slot = __ldg(a.slots + t);
        own = pages_to_score(a, slot, __ldg(a.positions + t), sel, true, lane, 32);
    }
    if (lane == 0) {
        owns[warp] = own;
        slot_of[warp] = slot;
    }
    for (int g = 0; g < a.grp; ++g) {
        float x[D / 32];
        load_query<T, D>(x, own ? a.q + t * a.q_tok + (h * a.grp + g) * a.q_head : nullptr, lane);
        const float unit = whole_query<T, D>(x, qpos + (g * N + warp) * D, qneg + (g * N + warp) * D, lane);
        if (lane == 0) qunit[g * N + warp] = unit;
    }
    __syncthreads();
    const int g = lane >> 2, tq = lane & 3;
    const signed char* ix = a.index + h * a.i_head;
    const int own0 = owns[2 * tq], own1 = owns[2 * tq + 1];
    // sequence by sequence: usually all eight stand in one
    for (int lead = 0; lead < N; ++lead) {
        if (!owns[lead]) continue;
        const int seq = slot_of[lead];
        int top = 0;
        bool first = true;
        for (int i = 0; i < N; ++i) {
            if (!owns[i] || slot_of[i] != seq) continue;
            if (i < lead) first = false;
            top = max(top, owns[i]);
        }
        if (!first) continue;
        const int lim0 = slot_of[2 * tq] == seq ? own0 : 0, lim1 = slot_of[2 * tq + 1] == seq ? own1 : 0;
        const int* row = a.table + seq * a.table_row;
        int next[UNROLL][2];
        auto look = [&](int j0) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int j = j0 + u * N * 16 + g + 8 * r;
                    next[u][r] = j < top ? __ldg(row + j) : -1;
                }
        };
        look(warp * 16);
#pragma unroll 1
        for (int j0 = warp * 16; j0 < top; j0 += N * 16 * UNROLL) {
            PageStep<D> st[UNROLL];
            int pid[UNROLL][2];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    pid[u][r] = next[u][r];
                    if (j0 + u * N * 16 + g + 8 * r < top && (pid[u][r] < 0 || pid[u][r] >= a.pages)) {
                        note_status(a.status, MQ_ERR_BAD_PAGE);
                        pid[u][r] = -1;
                    }
                }
                st[u].load(ix, a.i_page, pid[u], tq);
            }
            look(j0 + N * 16 * UNROLL);
            float best[UNROLL][4];   // page g: tokens 2 t, 2 t + 1; page g + 8
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) best[u][0] = best[u][1] = best[u][2] = best[u][3] = -INFINITY;
            for (int hd = 0; hd < a.grp; ++hd) {   // columns: one head of the 8 tokens
                int4 q[2 * D / 64];
#pragma unroll
                for (int b = 0; b < 2 * D / 64; ++b)
                    q[b] = *reinterpret_cast<const int4*>((b < D / 64 ? qpos : qneg) + (hd * N + g) * D + (b % (D / 64)) * 64 + 16 * tq);
                const float u0 = qunit[hd * N + 2 * tq], u1 = qunit[hd * N + 2 * tq + 1];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    int c[4];
                    st[u].dot(c, q);
#pragma unroll
                    for (int i = 0; i < 4; ++i) best[u][i] = fmaxf(best[u][i], (float)c[i] * (i & 1 ? u1 : u0));
                }
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int j = j0 + u * N * 16 + g + 8 * r;
                    if (j < lim0) keys[(long long)(2 * tq) * a.cols + j] = st[u].key(r, best[u][2 * r], pid[u][r] >= 0);
                    if (j < lim1) keys[(long long)(2 * tq + 1) * a.cols + j] = st[u].key(r, best[u][2 * r + 1], pid[u][r] >= 0);
                }
        }
    }
    __syncthreads();
    if (own) {
        choose<1>(keys + (long long)warp * a.cols, own, a.top_k - 1, sel, {hist[warp], list[warp], pick[warp], nullptr, nullptr}, 0, lane);
        if (lane == 0) sel[a.top_k - 1] = own;
    }
    if (!a.count || t >= a.n) return;
    __syncwarp();
    for (int k = lane; k < a.top_k; k += 32) {
        const int c = sel[k];   // listed: the slot and the column are in range
        int rank = -1;
        if (c >= 0) {
            const int pid = __ldg(a.table + slot * a.table_row + c);
            if (pid >= 0 && pid < a.pages) rank = (int)atomicAdd(a.count + (long long)h * a.pages + pid, 1u);
            else note_status(a.status, MQ_ERR_BAD_PAGE);
        }
        a.rank[((long long)t * a.hkv + h) * a.top_k + k] = rank;
    }
}

// ---- host ----------------------------------------------------------------------------------

PoolView view_of(const mq_paged_pool& p, int layer) {
    return {(const uint16_t*)p.k + layer * p.k_layer, (const uint16_t*)p.v + layer * p.v_layer, p.k_page, p.k_head,
            p.v_page, p.v_head, p.num_pages, p.page_size, __builtin_ctz((unsigned)p.page_size)};
}

// f(T{}, integral_constant<D>) for the pool's type and head_dim.
template <typename F>
int dispatch(int dtype, int D, F f) {
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (dtype == MQ_BF16) return D == 128 ? f(__nv_bfloat16{}, D128{}) : f(__nv_bfloat16{}, D64{});
    return D == 128 ? f(__half{}, D128{}) : f(__half{}, D64{});
}

void set_rt(RowArgs& a, bool eight) {
    a.rt = eight ? 8 : 16;
    a.rt_shift = eight ? 3 : 4;
}

// The choice kernel takes eight tokens to a CTA once that gives every SM a CTA of them and their keys fit (96 KB).
bool eight_fit(int n, int hkv, int D, int cols, int grp) {
    return (long long)n * hkv >= (long long)SEL_TOKENS * sm_count() && n >= SEL_TOKENS &&
           (D == 128 ? sel_eight_bytes<128>(cols, grp) : sel_eight_bytes<64>(cols, grp)) <= 98304;
}

// CTAs of the work line: two to an SM for head_dim 128 with 16 rows to an item (up to
// 255 registers a thread), three otherwise (168).  The rings take 64 KB of shared memory
// (head_dim 64: 32); with the schedule of a call near 2048 sequences and groups (48 KB)
// fewer fit, and the rest of the grid runs after them.
int row_grid(int D, int rt) { return sm_count() * (D == 128 && rt == 16 ? 2 : 3); }

// The page-by-page form's rounds: parts that stay in L2 from the kernel that writes them to the join.
constexpr size_t PART_BYTES = 96u << 20;
constexpr int BY_PAGE_TOKENS = 64;

// Tokens per round of the page-by-page form, or 0 where each token reads its own pages.  Page by page when
//  - there are more tokens than the table has slots, so that some stand in one sequence (150 / 250 tokens of one context of
//    16k: 47 / 61 us against 69 / 96; of 256 sequences with nothing in common: 237 against 216).  Which sequences a call
//    holds stands on the device, so tokens of one sequence in a table of more slots than the call has tokens stay with the
//    other form: the 69 / 96 us, and not the 237 for a decode batch,
//  - a page's keys and values are 16 times its parts for one token or more (500 tokens on two contexts of 16k, page
//    over group 64: 105 us against 202, 32: 107 against 205, 16: 204 against 216, 8: 378 against 235),
//  - the choice kernel takes eight tokens at a time (it counts for this form), a round holds 64 tokens or more, and
//    the pool has no more than 16 pages for each choice (the counts are cleared and read, 8 bytes a page).
int by_page_tokens(const mq_paged_sparse_params* p) {
    const mq_paged_pool& o = *p->pool;
    const int grp = p->num_q_heads / o.num_kv_heads, D = o.head_dim;
    const size_t part = 4 * (size_t)(D + 4), token = part * p->num_q_heads * p->top_k;
    const size_t most = PART_BYTES / token;
    if (most < BY_PAGE_TOKENS || p->n < BY_PAGE_TOKENS || o.page_size < 16 * grp || p->n <= p->num_slots) return 0;
    const int rounds = ceil_div(p->n, (int)(most < 0x7fffffff ? most : 0x7fffffff)), n = ceil_div(p->n, rounds);
    if (!eight_fit(n, o.num_kv_heads, D, p->table_cols, grp) || o.num_pages > 16ll * n * p->top_k) return 0;
    return n;
}

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// The prefixes go to the tensor-core kernel when a group has more rows than the
// 16 of a rows_kernel item on average, so that the row kernel would read the prefix
// more than once.  How long the prefix is stands on the device, so the rule cannot
// look at it; tensor cores against rows for one group of two q heads per kv head,
// 8 kv heads x 128, own parts of 100 (us a call):
//   behind      64          1k          8k          32k         128k
//    9 seqs  23.2 / 14.3  22.2 / 15.9  23.8 / 21.8  46 / 48    125 / 173
//   32 seqs  24.3 / 15.8  23.1 / 17.2  31.4 / 30.9  50 / 83    133 / 340
//   64 seqs  25.7 / 17.2  24.0 / 21.5  35.1 / 48.0  57 / 155   142 / 528
// (A scale of zero stays out: there a masked score of minus infinity would not stay one.)
bool tc_prefix(long long tokens, int grp, int NG, float scale) {
    return NG > 0 && NG <= PFX_MAX_GROUPS && tokens * grp > 16ll * NG && scale != 0.f;
}

struct Shape {
    int D, hq;
    long long tokens;
    bool attend, groups, tc;
};

size_t row_workspace(const Shape& s, WsView* v, void* base) {
    size_t o = 256;
    auto take = [&](size_t bytes) {
        const size_t at = o;
        o += up256(bytes);
        return at;
    };
    const size_t rows = (size_t)s.tokens * s.hq * (s.D + 4) * 4;
    const size_t tok = take(s.attend ? (size_t)s.tokens * sizeof(TokInfo) : 0);
    const size_t own = take(s.groups ? rows : 0);
    const size_t slots = take((size_t)2 * row_grid(s.D, 8) * ROW_WARPS * MAX_RT * (s.D + 4) * 4);
    const size_t pfx = take(s.groups ? (s.tc ? 2 * rows : rows) : 0);
    const size_t pfx_slots = take(s.tc ? (size_t)2 * sm_count() * PROWS * (s.D + 4) * 4 : 0);
    if (v) {
        uint8_t* b = (uint8_t*)base;
        v->head = (uint32_t*)b;
        v->tok = (TokInfo*)(b + tok);
        v->own_rowp = (float*)(b + own);
        v->slots = (float*)(b + slots);
        v->pfx_rowp = (float*)(b + pfx);
        v->pfx_slots = (float*)(b + pfx_slots);
    }
    return o;
}

size_t by_page_workspace(const mq_paged_sparse_params* p, int n, ByPage* v, void* base) {
    const size_t bins = (size_t)p->pool->num_kv_heads * p->pool->num_pages;
    const size_t entries = (size_t)n * p->pool->num_kv_heads * p->top_k;
    const size_t off = up256(16 + bins * 4), items = off + up256(bins * 4), list = items + up256(entries * 16);
    const size_t rank = list + up256(entries * 16), parts = rank + up256(entries * 4);
    if (v) {
        uint8_t* b = (uint8_t*)base;
        v->cursor = (unsigned long long*)b;
        v->count = (uint32_t*)(b + 16);
        v->off = (uint32_t*)(b + off);
        v->items = (int4*)(b + items);
        v->list = (int4*)(b + list);
        v->rank = (int*)(b + rank);
        v->parts = (float*)(b + parts);
        v->per_item = 8 * BY_PAGE_NT / (p->num_q_heads / p->pool->num_kv_heads);
    }
    return parts + (size_t)n * p->num_q_heads * p->top_k * (p->pool->head_dim + 4) * 4;
}

Shape shape_of(const mq_paged_attend_params* p) {
    return {p->pool->head_dim, p->num_q_heads, p->total_q, true, p->num_groups > 0,
            tc_prefix(p->total_q, p->num_q_heads / p->pool->num_kv_heads, p->num_groups, p->scale)};
}
Shape shape_of(const mq_paged_sparse_params* p) {
    return {p->pool->head_dim, p->num_q_heads, p->n, false, false, false};
}

// A layer's K or V as a rank-5 map of boxes of `rows` rows of a page, `blocks` blocks of 64 channels.
bool pool_map(CUtensorMap* m, const mq_paged_pool& p, const void* base, long long page, long long head, int rows, int blocks) {
    const cuuint64_t row = (cuuint64_t)p.head_dim * 2, block = row * p.page_size;
    const cuuint64_t dims[5] = {64, (cuuint64_t)p.page_size, (cuuint64_t)p.head_dim / 64, (cuuint64_t)p.num_kv_heads, (cuuint64_t)p.num_pages};
    // the stride of a dimension of one is never used and may be anything
    const cuuint64_t strides[4] = {row, 128, p.num_kv_heads > 1 ? (cuuint64_t)head * 2 : block, p.num_pages > 1 ? (cuuint64_t)page * 2 : block};
    const cuuint32_t box[5] = {64, (cuuint32_t)rows, (cuuint32_t)blocks, 1, 1};
    return make_tmap_nd(m, base, p.dtype == MQ_BF16, 5, dims, strides, box);
}
bool pool_maps(CUtensorMap* k, CUtensorMap* v, const mq_paged_pool& p, const PoolView& at, int rows, int blocks) {
    return pool_map(k, p, at.k, at.k_page, at.k_head, rows, blocks) && pool_map(v, p, at.v, at.v_page, at.v_head, rows, blocks);
}

template <typename T, int D>
int run_prefix(const RowArgs& a, const mq_paged_pool& pool, cudaStream_t st) {
    CUtensorMap tk, tv;
    if (!pool_maps(&tk, &tv, pool, a.pool, pool.page_size, 1)) return MQ_ERR_CUDA;
    auto kernel = prefix_kernel<T, D>;
    const size_t smem = PfxSmem<D>::bytes(a.NG);
    static SmemLimit limit;
    cudaError_t e = allow_smem(kernel, smem, limit);
    if (e == cudaSuccess) e = launch(kernel, dim3(sm_count()), dim3(PFX_THREADS), smem, st, tk, tv, a);
    return e == cudaSuccess ? MQ_OK : note_cuda(e, "paged prefix attention");
}

template <typename T, int D, int MODE>
cudaError_t run_join(const RowArgs& a, uint32_t row_warps, cudaStream_t st) {
    const long long rows = (long long)a.total_q * a.hq;
    // As many warps to a row as leave all CTAs resident at once (three to an SM): a second wave costs more
    // than the warps save (1024 rows of 34 parts, 512 CTAs: 14 us).
    auto join = [&](auto split) {
        constexpr int S = decltype(split)::value;
        return launch(join_kernel<T, D, MODE, S>, dim3((unsigned)((rows * S + 7) / 8)), dim3(256), 0, st, a, row_warps);
    };
    const long long room = 3ll * sm_count() * 8 / rows;   // warps to a row
    return room >= 8   ? join(std::integral_constant<int, 8>{})
           : room >= 4 ? join(std::integral_constant<int, 4>{})
           : room >= 2 ? join(std::integral_constant<int, 2>{})
                       : join(std::integral_constant<int, 1>{});
}

template <typename T, int D, int MODE, int NT>
int run_rows(const RowArgs& a, const mq_paged_pool& pool, cudaStream_t st) {
    CUtensorMap tk, tv;
    if (!pool_maps(&tk, &tv, pool, a.pool, GRP, D / 64)) return MQ_ERR_CUDA;
    auto kernel = rows_kernel<T, D, MODE, NT>;
    const size_t smem = (size_t)ROW_WARPS * RowWarp<T, D, NT>::RING + 1024 + (MODE == 0 ? sched_bytes(a.B, a.NG) : 0);
    static SmemLimit limit;
    cudaError_t e = allow_smem(kernel, smem, limit);
    if (e != cudaSuccess) return note_cuda(e, "paged attention attribute");
    const int grid = row_grid(D, 8 * NT);
    e = launch(kernel, dim3(grid), dim3(ROW_THREADS), smem, st, tk, tv, a);
    if (e == cudaSuccess) e = run_join<T, D, MODE>(a, (uint32_t)grid * ROW_WARPS, st);
    return e == cudaSuccess ? MQ_OK : note_cuda(e, "paged attention");
}

template <typename T, int D>
int run_attend(const RowArgs& a, const mq_paged_pool& pool, cudaStream_t st) {
    if (a.tc) {
        const int rc = run_prefix<T, D>(a, pool, st);
        if (rc) return rc;
    }
    return a.rt == 8 ? run_rows<T, D, 0, 1>(a, pool, st) : run_rows<T, D, 0, 2>(a, pool, st);
}

// After the choice, whose counts are in place.
template <typename T, int D>
int run_by_page(const RowArgs& a, const mq_paged_pool& pool, cudaStream_t st) {
    CUtensorMap tk, tv;
    if (!pool_maps(&tk, &tv, pool, a.pool, GRP, D / 64)) return MQ_ERR_CUDA;
    auto kernel = by_page_kernel<T, D>;
    const size_t smem = (size_t)ROW_WARPS * RowWarp<T, D, BY_PAGE_NT>::RING + 1024;
    static SmemLimit limit;
    cudaError_t e = allow_smem(kernel, smem, limit);
    const long long bins = (long long)a.hkv * a.pool.pages, entries = (long long)a.total_q * a.hkv * a.top_k;
    if (e == cudaSuccess) e = launch(plan_kernel, dim3((unsigned)((bins + 255) / 256)), dim3(256), 0, st, a.bp, a.hkv, a.pool.pages);
    if (e == cudaSuccess) e = launch(list_kernel, dim3((unsigned)((entries + 255) / 256)), dim3(256), 0, st, a);
    if (e == cudaSuccess) e = launch(kernel, dim3(row_grid(D, 8 * BY_PAGE_NT)), dim3(ROW_THREADS), smem, st, tk, tv, a);
    if (e == cudaSuccess) e = run_join<T, D, 2>(a, 0, st);
    return e == cudaSuccess ? MQ_OK : note_cuda(e, "paged attention by page");
}

bool q_ok(const void* q, long long tok, long long head) {
    return q && (reinterpret_cast<uintptr_t>(q) & 15) == 0 && tok % 8 == 0 && head % 8 == 0;
}

template <typename T, int D>
int run_select(const SelArgs& s, cudaStream_t st) {
    const long long items = (long long)s.n * s.hkv;
    if (s.count || eight_fit(s.n, s.hkv, D, s.cols, s.grp)) {   // (page by page: whatever a last round has left)
        static SmemLimit limit;
        const size_t smem = sel_eight_bytes<D>(s.cols, s.grp);
        cudaError_t e = allow_smem(select_eight_kernel<T, D>, smem, limit);
        if (e == cudaSuccess)
            e = launch(select_eight_kernel<T, D>, dim3((unsigned)ceil_div(s.n, SEL_TOKENS) * s.hkv), dim3(SEL_TOKENS * 32), smem, st, s);
        return e == cudaSuccess ? MQ_OK : note_cuda(e, "page selection");
    }
    static SmemLimit limit;
    const size_t smem = sel_one_bytes<D>(s.cols, s.grp);
    cudaError_t e = allow_smem(select_one_kernel<T, D>, smem, limit);
    if (e != cudaSuccess) return note_cuda(e, "page selection attribute");
    // a cluster to an item: doubled while all its CTAs have an SM each and a CTA keeps 256 pages or more
    unsigned ranks = 1;
    while (ranks < 8 && items * ranks * 2 <= sm_count() && s.cols >= 512 * (int)ranks) ranks *= 2;
    e = launch_cluster(select_one_kernel<T, D>, (unsigned)items * ranks, ranks, dim3(SEL_WARPS * 32), smem, st, s);
    return e == cudaSuccess ? MQ_OK : note_cuda(e, "page selection");
}

}  // namespace paged
}  // namespace mq

using namespace mq::paged;

extern "C" {

size_t mq_paged_attend_workspace_bytes(const mq_paged_attend_params* p) {
    if (!p || !p->pool || p->total_q < 0 || p->pool->num_kv_heads < 1) return 0;
    return row_workspace(shape_of(p), nullptr, nullptr);
}

int mq_paged_attend(const mq_paged_attend_params* p, cudaStream_t st) {
    if (!p || !pool_ok(p->pool) || p->num_seqs < 0 || p->num_seqs > MAX_SEQS || p->total_q < 0 || p->num_groups < 0 ||
        p->num_groups > p->num_seqs || p->num_q_heads < 1 || p->num_q_heads % p->pool->num_kv_heads || p->layer < 0 ||
        p->layer >= p->pool->num_layers || p->num_slots < 1 || p->table_cols < 1 ||
        (!p->q_starts && p->num_seqs != p->total_q) || (p->num_groups && (!p->group_starts || !p->prefix_pages)))
        return MQ_ERR_INVALID_ARGUMENT;
    if (!p->total_q || !p->num_seqs) return p->total_q ? MQ_ERR_INVALID_ARGUMENT : MQ_OK;
    if (!q_ok(p->q, p->q_token, p->q_head) || !p->out || (reinterpret_cast<uintptr_t>(p->out) & 15) || !p->table ||
        !p->lengths || !p->slots || (long long)p->total_q * p->num_q_heads > 0x7fffffffll)
        return MQ_ERR_INVALID_ARGUMENT;
    if (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 255) ||
        p->workspace_bytes < mq_paged_attend_workspace_bytes(p))
        return MQ_ERR_WORKSPACE;
    RowArgs a = {};
    a.pool = view_of(*p->pool, p->layer);
    a.q = (const uint16_t*)p->q;
    a.q_tok = p->q_token;
    a.q_head = p->q_head;
    a.out = (uint16_t*)p->out;
    a.table = p->table;
    a.table_row = p->table_row;
    a.num_slots = p->num_slots;
    a.cols = p->table_cols;
    a.lengths = p->lengths;
    a.slots = p->slots;
    a.q_starts = p->q_starts;
    a.group_starts = p->group_starts;
    a.prefix_pages = p->prefix_pages;
    a.B = p->num_seqs;
    a.NG = p->num_groups;
    a.total_q = p->total_q;
    a.hq = p->num_q_heads;
    a.hkv = p->pool->num_kv_heads;
    a.grp = a.hq / a.hkv;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.status = p->status;
    const Shape s = shape_of(p);
    row_workspace(s, &a.ws, p->workspace);
    a.tc = s.tc;
    // 8 rows to an item when a sequence (and a group whose prefix is not on the tensor-core kernel) has no
    // more on average: half the tensor work a group; otherwise 16, so that the keys are read half as often
    const long long rows = (long long)a.total_q * a.grp;
    set_rt(a, rows <= 8ll * a.B && (!a.NG || a.tc || rows <= 8ll * a.NG));
    return dispatch(p->pool->dtype, s.D, [&](auto T, auto D) { return run_attend<decltype(T), decltype(D)::value>(a, *p->pool, st); });
}

size_t mq_paged_sparse_workspace_bytes(const mq_paged_sparse_params* p) {
    if (!p || !p->pool || p->n < 0 || p->pool->num_kv_heads < 1 || p->num_q_heads < p->pool->num_kv_heads || p->top_k < 1) return 0;
    const int n = by_page_tokens(p);
    return n ? by_page_workspace(p, n, nullptr, nullptr) : row_workspace(shape_of(p), nullptr, nullptr);
}

int mq_paged_sparse(const mq_paged_sparse_params* p, cudaStream_t st) {
    if (!p || !pool_ok(p->pool) || !p->pool->index || p->n < 0 || p->num_q_heads < 1 ||
        p->num_q_heads % p->pool->num_kv_heads || p->num_q_heads / p->pool->num_kv_heads > MAX_SPARSE_GROUP || p->layer < 0 ||
        p->layer >= p->pool->num_layers || p->num_slots < 1 || p->table_cols < 1 || p->table_cols > MAX_SPARSE_COLS ||
        p->top_k < 1 || p->top_k > MAX_SPARSE_COLS || (long long)p->n * p->num_q_heads > 0x7fffffffll)
        return MQ_ERR_INVALID_ARGUMENT;
    if (!p->n) return MQ_OK;
    // the work line is counted in 31 bits
    if ((long long)p->n * p->pool->num_kv_heads * ceil_div(p->num_q_heads / p->pool->num_kv_heads, 8) *
            ((long long)p->top_k * (p->pool->page_size / GRP) + ITEM_UNITS) > 0x7fffffffll)
        return MQ_ERR_INVALID_ARGUMENT;
    if (!q_ok(p->q, p->q_token, p->q_head) || !p->out || (reinterpret_cast<uintptr_t>(p->out) & 15) || !p->selected ||
        !p->table || !p->slots || !p->positions)
        return MQ_ERR_INVALID_ARGUMENT;
    if (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 255) ||
        p->workspace_bytes < mq_paged_sparse_workspace_bytes(p))
        return MQ_ERR_WORKSPACE;
    const mq_paged_pool& o = *p->pool;
    SelArgs s = {};
    s.index = o.index + p->layer * o.i_layer;
    s.i_page = o.i_page;
    s.i_head = o.i_head;
    s.q = (const uint16_t*)p->q;
    s.q_tok = p->q_token;
    s.q_head = p->q_head;
    s.table = p->table;
    s.table_row = p->table_row;
    s.slots = p->slots;
    s.positions = p->positions;
    s.selected = p->selected;
    s.num_slots = p->num_slots;
    s.cols = p->table_cols;
    s.pages = o.num_pages;
    s.n = p->n;
    s.shift = __builtin_ctz((unsigned)o.page_size);
    s.hkv = o.num_kv_heads;
    s.grp = p->num_q_heads / o.num_kv_heads;
    s.top_k = p->top_k;
    s.status = p->status;
    RowArgs a = {};
    a.pool = view_of(o, p->layer);
    a.q = s.q;
    a.q_tok = p->q_token;
    a.q_head = p->q_head;
    a.out = (uint16_t*)p->out;
    a.table = p->table;
    a.table_row = p->table_row;
    a.num_slots = p->num_slots;
    a.cols = p->table_cols;
    a.slots = p->slots;
    a.positions = p->positions;
    a.selected = p->selected;
    a.total_q = p->n;
    a.hq = p->num_q_heads;
    a.hkv = o.num_kv_heads;
    a.grp = a.hq / a.hkv;
    a.top_k = p->top_k;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.status = p->status;
    set_rt(a, a.grp <= 8);
    const int round = by_page_tokens(p);
    if (round) by_page_workspace(p, round, &a.bp, p->workspace);
    else row_workspace(shape_of(p), &a.ws, p->workspace);
    for (long long t0 = 0; t0 < p->n; t0 += round ? round : p->n) {
        s.n = a.total_q = round ? (int)std::min<long long>(round, p->n - t0) : p->n;
        s.q = a.q = (const uint16_t*)p->q + t0 * p->q_token;
        a.out = (uint16_t*)p->out + t0 * a.hq * o.head_dim;
        a.selected = s.selected = p->selected + t0 * a.hkv * a.top_k;
        a.slots = s.slots = p->slots + t0;
        a.positions = s.positions = p->positions + t0;
        if (round) {
            s.count = a.bp.count;
            s.rank = a.bp.rank;
            const long long words = (16 + (long long)a.hkv * o.num_pages * 4 + 15) / 16;
            const long long blocks = (words + 255) / 256, most = 2ll * sm_count();
            const cudaError_t e = launch(clear_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st,
                                         reinterpret_cast<uint4*>(a.bp.cursor), words);
            if (e != cudaSuccess) return mq::note_cuda(e, "paged attention by page");
        }
        const int rc = dispatch(o.dtype, o.head_dim, [&](auto T, auto D) {
            using E = decltype(T);
            constexpr int d = decltype(D)::value;
            const int r = run_select<E, d>(s, st);
            if (r) return r;
            if (round) return run_by_page<E, d>(a, o, st);
            return a.rt == 8 ? run_rows<E, d, 1, 1>(a, o, st) : run_rows<E, d, 1, 2>(a, o, st);
        });
        if (rc) return rc;
    }
    return MQ_OK;
}

}  // extern "C"
