// A token for each row of logits: temperature, top-k, top-p and min-p, drawn
// with a given number per row.
//
// Mathematics: w_i = 2^((l_i - max) log2(e) / T).  Tokens in descending order of
// their logit, equal ones in ascending order of their number; the first top_k
// stay; of those the ones before which less than top_p of their sum lies; of
// those the ones with w >= min_p.  The token is the first, in ascending order of
// the number, up to which the sum of what stays exceeds u times its total.
//
// Every one of these is a border between tokens, so the answer has to be that of
// the definition and not of an order of sums: a token's place in the order is a
// whole number (its logit's bits, made to ascend, over its number turned
// around), and its weight is computed in 64 bits and held as a multiple of
// 2^-43, so that sums are exact, in any order, up to 2^20 tokens.  In 32 bits a
// flat row of 152k tokens would get another token once in a hundred draws.
//
// HBM reads the row once, 4 or 2 bytes a token; what is done with it costs more.  A cluster of up to 8 CTAs takes a row,
// each a contiguous share of it, and keeps it in shared memory as fp32 where it fits.  What follows depends on the rules:
//   a top_k of up to FEW: the top_k-th largest of the threads' own maxima is a bound
//     that top_k tokens reach; the few hundred that do go to the first CTA, which
//     does the rest alone, in descending order and then by number;
//   top_p alone: a histogram of the logits beside the sum of all weights tells which
//     bins the border can lie in; the tokens of those, and the sums of the tokens
//     above them by pieces of the row, go to the first CTA, which finds the border and
//     the token in its piece while the others make room for the next row;
//   neither: sums of pieces of the row, in the order of the tokens.
// Rows that do not fit these (thousands of equal logits at a border, a large top_k) take the general form: a histogram
// with exact sums for each border, refined until the border's bin can be sorted.
//
// Bound: latency for one row (14 us of 152k tokens: five meetings of the cluster of 1 to 2 us each, the first CTA's steps);
// for many, a nucleus is a chain per row of load, histogram, sums, sort, on two CTAs an SM: 256 rows of 152k in 16 bits
// 309 us (0.25 TB/s), 64 rows with rules of their own, fp32, 80 us (0.48 TB/s).  Profiled, the 256 rows: issue slots 55 %
// busy, 64-bit floating point 16 %, integers 48 %, 27 % of the warps' time in barriers.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_common.cuh"

namespace mq {
namespace sampling {

using paged::allow_smem;
using paged::ceil_div;
using paged::cluster_rank;
using paged::cluster_size;
using paged::launch_cluster;
using paged::SmemLimit;
using paged::sm_count;

using u64 = unsigned long long;

constexpr int NT = 512, NW = NT / 32;
constexpr int BINS = 2048;          // four to a thread
constexpr int CAP = 2048;           // tokens that are sorted
constexpr int FEW = 1024;           // the largest top_k whose tokens one CTA takes
constexpr int MAX_RANKS = 8;
constexpr int TABLE = 128;          // of 2^(j / TABLE)
constexpr int FRAC = 43;            // a weight of 1 is 2^43
constexpr double ONE = 8796093022208.0;
constexpr int MAX_VOCAB = 1 << 20;  // a row's sum stays below 2^63
constexpr float COUNT_SPAN = 40.f;  // logits below the maximum that the histogram of a count spreads over its bins
constexpr double MASS_SPAN = 20.0;  // octaves below the maximum that the histogram of a mass spreads over its bins

struct Args {
    const void* logits;
    long long row;        // elements between rows
    int n, vocab, share;  // share: tokens to a CTA
    const float* u;
    const float* temperature;   // per row, or null for the value
    const int* top_k;
    const float* top_p;
    const float* min_p;
    float temperature_v, top_p_v, min_p_v;
    int top_k_v;
    int* out;
};

// Two 16-bit values of a word (no word holds two of fp32, and none is asked for).
template <typename T>
__device__ __forceinline__ float2 two_up(uint32_t w) {
    if (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    return make_float2(bf16lo(w), bf16hi(w));
}

template <typename T>
__device__ __forceinline__ float load_one(const T* p) {
    if (sizeof(T) == 4) return __ldg(reinterpret_cast<const float*>(p));
    return two_up<T>(__ldg(reinterpret_cast<const unsigned short*>(p))).x;
}

__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ u64 place_key(float x, int token) { return (u64)order_key(x) << 32 | (uint32_t)~token; }
__device__ __forceinline__ int token_of(u64 key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float logit_of(u64 key) {
    const uint32_t k = (uint32_t)(key >> 32);
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The cluster's barrier, for warps whose threads may come to it one by one (loops and branches lie before it).
__device__ __forceinline__ void cluster_meet() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Remote shared memory of the cluster.
__device__ __forceinline__ uint32_t peer(const void* p, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ void peer_st(uint32_t at, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}
__device__ __forceinline__ uint4 peer_ld4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t peer_ld(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t peer_add(uint32_t at, uint32_t v) {
    uint32_t old;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(at), "r"(v) : "memory");
    return old;
}

// What a CTA needs beside its share of the row.
struct Shared {
    uint32_t count[BINS];             // of this CTA
    union {                           // the bins' sums are read before tokens are listed
        struct {
            uint32_t low[BINS], high[BINS];   // of its weights
        };
        u64 list[CAP];
    };
    u64 slot[2][MAX_RANKS][4];        // what the CTAs tell each other, two turns of it
    u64 warp_sum[NW];
    u64 found[4];
    double two_to[TABLE];             // 2^(j / TABLE)
    u64 pieces[MAX_RANKS * NW];       // sums of the warps' pieces of the row, in the first CTA
    u64 ends[2 * NW];                 // the warps' smallest and largest keys
    int taken;
};

// The row's weights.  2^y by a table of 2^(j / 128) and the Taylor polynomial of 2^(r / 128), |r| <= 1 / 2, up to r^4 (the
// next term is below 2^-49).
struct Weight {
    double scale, top;   // 128 log2(e) / T; the maximum
    float max;
    __device__ __forceinline__ double place(float l) const {   // 128 y
        const double d = ((double)l - top) * scale;
        return l == max ? 0.0 : d;
    }
    // 2^(z / 128), z <= 0, at least 2^-1000
    __device__ __forceinline__ double as_double(double z, const double* two_to) const {
        z = z > -1000.0 * TABLE ? z : -1000.0 * TABLE;
        constexpr double MAGIC = 6755399441055744.0;   // 1.5 x 2^52: rounds to whole numbers
        const double t = z + MAGIC, r = z - (t - MAGIC);
        const int n = __double2loint(t);
        double p = 3.583032305400251e-11;              // (ln(2) / 128)^k / k!
        p = fma(p, r, 2.6466421444330967e-08);
        p = fma(p, r, 1.4662262387640423e-05);
        p = fma(p, r, 5.4152123481245725e-03);
        p = fma(p, r, 1.0) * two_to[n & (TABLE - 1)];
        return __hiloint2double(__double2hiint(p) + (n >> 7) * (1 << 20), __double2loint(p));
    }
    // in multiples of 2^-43, rounded to the nearest: the last place of numbers from 2^9 to 2^10
    __device__ __forceinline__ u64 of(double z, const double* two_to) const {
        static_assert(FRAC == 43, "the last place of 2^9");
        return (u64)__double_as_longlong(as_double(z, two_to) + 512.0) - (u64)0x4080000000000000ull;
    }
    __device__ __forceinline__ u64 of(float l, const double* two_to) const { return of(place(l), two_to); }
};

// Exclusive sum over the CTA's threads; total for every thread.
template <typename V>
__device__ __forceinline__ V block_scan(V v, u64* sm, V* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) sm[warp] = x;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const V s = (V)sm[w];
        if (w < warp) before += s;
        all += s;
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

__device__ __forceinline__ int block_sum_of(int v, u64* sm) {
    v = (int)__reduce_add_sync(0xffffffffu, (unsigned)v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = (u64)v;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < NW; ++w) all += (int)sm[w];
    __syncthreads();
    return all;
}
// The same for an estimate.
__device__ __forceinline__ double block_scan_double(double v, double* sm, double* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sm[warp] = x;
    __syncthreads();
    double before = 0, all = 0;
    for (int w = 0; w < NW; ++w) {
        if (w < warp) before += sm[w];
        all += sm[w];
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

// list[0 .. n - 1] in descending order, n <= CAP; the places up to the next power of two are filled with 0.
__device__ __forceinline__ void sort_down(u64* list, int n) {
    int size = 32;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += NT) list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = threadIdx.x; i < size / 2; i += NT) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;   // a has bit j clear
                const u64 x = list[a], y = list[b];
                if ((x < y) == ((a & k) == 0)) {
                    list[a] = y;
                    list[b] = x;
                }
            }
            __syncthreads();
        }
}

template <typename T, bool NEAR>   // NEAR: the share of the row stays in shared memory
__global__ void __launch_bounds__(NT, 2) sample_kernel(const Args a) {
    extern __shared__ __align__(16) uint8_t sample_raw[];
    Shared& s = *reinterpret_cast<Shared*>(sample_raw);
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ranks = (int)cluster_size(), rank = (int)cluster_rank();
    const int r = blockIdx.x / ranks;
    const T* row = reinterpret_cast<const T*>(a.logits) + (long long)r * a.row;
    const int lo = min(a.vocab, rank * a.share), n = min(a.vocab, lo + a.share) - lo;
    const T* x = row + lo;
    if (tid < TABLE) s.two_to[tid] = exp2((double)tid / TABLE);
    if (tid == 0) s.taken = 0;
    // the share, 16 bytes at a time; in shared memory it lies as in global memory to 16 bytes, with minus infinity before
    // and behind
    float best = -INFINITY, least = INFINITY;
    int best_at = 0;
    auto look = [&](float v, int i) {
        if (v > best) best = v, best_at = i;   // (a thread's tokens ascend: the first of equal ones)
        if (v > -INFINITY) least = fminf(least, v);
    };
    auto clean = [](float v) { return v == v ? v + 0.f : -INFINITY; };   // NaN is never drawn; -0 is 0
    constexpr int PER = 16 / sizeof(T);
    const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));   // elements past a 16-byte border
    float* near = reinterpret_cast<float*>(sample_raw + ((sizeof(Shared) + 15) & ~(size_t)15));
    const int quads = (off + n + 3) / 4;
    {
        const int head = min(n, off ? PER - off : 0), body = (n - head) / PER, tail = n - head - body * PER;
        if (NEAR) {
            if (tid < off) near[tid] = -INFINITY;
            if (tid < 4 && off + n + tid < 4 * quads) near[off + n + tid] = -INFINITY;
        }
        if (tid < head) {
            const float v = clean(load_one(x + tid));
            look(v, tid);
            if (NEAR) near[off + tid] = v;
        }
        const uint4* from = reinterpret_cast<const uint4*>(x + head);
        float4* to = reinterpret_cast<float4*>(near + (off ? PER : 0));
        constexpr int DEEP = 4;
        for (int i0 = tid; i0 < body; i0 += NT * DEEP) {
            uint4 v[DEEP];
#pragma unroll
            for (int k = 0; k < DEEP; ++k)
                if (i0 + k * NT < body) v[k] = __ldg(from + i0 + k * NT);
#pragma unroll
            for (int k = 0; k < DEEP; ++k) {
                const int i = i0 + k * NT;
                if (i >= body) break;
                const uint32_t e[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
                float f[PER];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (PER == 4) {
                        f[c] = clean(__uint_as_float(e[c]));
                    } else {
                        const float2 a = two_up<T>(e[c]);
                        f[2 * c % PER] = clean(a.x);
                        f[(2 * c + 1) % PER] = clean(a.y);
                    }
                }
#pragma unroll
                for (int c = 0; c < PER; ++c) look(f[c], head + i * PER + c);
                if (NEAR) {
#pragma unroll
                    for (int c = 0; c < PER; c += 4) to[i * (PER / 4) + c / 4] = make_float4(f[c], f[c + 1], f[c + 2], f[c + 3]);
                }
            }
        }
        if (tid < tail) {
            const int i = head + body * PER + tid;
            const float v = clean(load_one(x + i));
            look(v, i);
            if (NEAR) near[off + i] = v;
        }
    }
    const float own_best = best;   // this thread's
    auto at = [&](int i) -> float { return NEAR ? near[off + i] : clean(load_one(x + i)); };
    // Places 4 j .. 4 j + 3 of the share, of which the first `off` lie before it: minus infinity there and behind the end.
    auto quad = [&](int j) -> float4 {
        if (NEAR) return reinterpret_cast<const float4*>(near)[j];
        const int i = 4 * j - off;
        if (i >= 0 && i + 4 <= n) {
            if (sizeof(T) == 4) {
                const float4 q = __ldg(reinterpret_cast<const float4*>(x + i));
                return make_float4(clean(q.x), clean(q.y), clean(q.z), clean(q.w));
            }
            const uint2 q = __ldg(reinterpret_cast<const uint2*>(x + i));
            const float2 a = two_up<T>(q.x), b = two_up<T>(q.y);
            return make_float4(clean(a.x), clean(a.y), clean(b.x), clean(b.y));
        }
        auto one = [&](int k) { return i + k >= 0 && i + k < n ? clean(load_one(x + i + k)) : -INFINITY; };
        return make_float4(one(0), one(1), one(2), one(3));
    };
    auto own_quad = [&](int j, int end) { return j < end ? quad(j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); };
    // f(logit, place in the share) for every token, four of a thread at a time, where any of a warp's is `low` or more; by
    // whole warps, with minus infinity where there is none
    auto each = [&](float low, auto f) {
        float4 next = own_quad(warp * 32 + lane, quads);
        for (int j0 = warp * 32; j0 < quads; j0 += NT) {
            const int j = j0 + lane;
            const float4 q = next;
            next = own_quad(j + NT, quads);   // on its way while this one is worked on
            if (!__any_sync(0xffffffffu, fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)) >= low)) continue;
            const int i = 4 * j - off;
            f(q.x, i);
            f(q.y, i + 1);
            f(q.z, i + 2);
            f(q.w, i + 3);
        }
    };
    int turn = 0;
    // every CTA's four words to every CTA, all threads' writes before visible to all
    auto tell = [&](u64 v0, u64 v1, u64 v2, u64 v3) {   // the values of thread 0
        if (tid == 0) s.found[0] = v0, s.found[1] = v1, s.found[2] = v2, s.found[3] = v3;
        __syncthreads();
        turn ^= 1;
        if (tid < 4 * ranks) peer_st(peer(&s.slot[turn][rank][tid & 3], tid >> 2), s.found[tid & 3]);
        cluster_meet();
    };
    u64 first;   // the largest logit, the first of equal ones
    {   // the maximum and the smallest finite logit
        u64 b = place_key(best, lo + best_at);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
            least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
        }
        if (lane == 0) {
            s.warp_sum[warp] = b;
            s.list[warp] = order_key(least);
        }
        __syncthreads();
        u64 l = ~0ull;
        b = 0;
        for (int w = 0; w < NW; ++w) {
            b = max(b, s.warp_sum[w]);
            l = min(l, s.list[w]);
        }
        if (ranks > 1) cluster_meet();   // every CTA runs: its shared memory may be written
        tell(b, l, 0, 0);
        first = 0;
        l = ~0ull;
        for (int c = 0; c < ranks; ++c) {
            first = max(first, s.slot[turn][c][0]);
            l = min(l, s.slot[turn][c][1]);
        }
        least = logit_of(l << 32);
    }
    const float top = logit_of(first);
    const float temp = a.temperature ? __ldg(a.temperature + r) : a.temperature_v;
    if (!(temp > 0.f) || top == -INFINITY) {   // all CTAs alike
        if (rank == 0 && tid == 0) a.out[r] = top == -INFINITY ? -1 : token_of(first);
        return;
    }
    const int top_k = a.top_k ? __ldg(a.top_k + r) : a.top_k_v;
    const float top_p = a.top_p ? __ldg(a.top_p + r) : a.top_p_v;
    const float min_p = a.min_p ? __ldg(a.min_p + r) : a.min_p_v;
    const float u = __ldg(a.u + r);
    const bool by_count = top_k > 0 && top_k < a.vocab, by_mass = top_p < 1.f;
    const Weight w = {TABLE * 1.4426950408889634 / (double)temp, (double)top, top};
    const double floor_z = min_p > 0.f ? TABLE * log2((double)fminf(min_p, 1.f)) : -INFINITY;   // w >= min_p: 128 y from here on
    // the first sum in units of 2^-43 that exceeds u times the total
    auto aim = [&](u64 total) -> u64 {
        const double x = (u > 0.f ? (double)u : 0.0) * (double)total;   // (NaN counts as 0)
        return x < (double)total ? min((u64)x, total - 1) : total - 1;
    };
    // bins of equal width in the logit, from the maximum down
    float fine = 0.f, span = 0.f;
    auto spread = [&](float most) {
        span = fminf(fminf(top - least, most), 3.402823466e38f);   // (of a number: past it lies the last bin)
        fine = span > 0.f ? (float)BINS / span : 0.f;
    };
    auto bin_of = [&](float l) -> int {
        // a whole number by adding 2^23 (an int conversion takes four times as long); past 2^23 + BINS - 1 the last bin, as
        // minus infinity; below 2^23 (a quarter of a bin from the maximum) the first; the maximum at +infinity would be NaN
        const float d = fmaxf(fminf(fmaf(top - l, fine, 8388607.5f), 8388608.f + (float)(BINS - 1)), 8388608.f);
        return l == top ? 0 : (int)(__float_as_uint(d) & 0x7fffffu);
    };
    const float mass_span = (float)(MASS_SPAN * TABLE / w.scale);
    // every CTA's counts of this thread's four bins
    auto sum_bins = [&](uint32_t (&c4)[4]) {
        c4[0] = c4[1] = c4[2] = c4[3] = 0;
        for (int c = 0; c < ranks; ++c) {
            const uint4 q = peer_ld4(peer(&s.count[4 * tid], c));
            c4[0] += q.x, c4[1] += q.y, c4[2] += q.z, c4[3] += q.w;
        }
    };
    // a token into the first CTA's list, by whole warps; what does not fit is counted all the same
    auto hand_in = [&](bool take, u64 key) {
        const unsigned who = __ballot_sync(0xffffffffu, take);
        if (!who) return;
        uint32_t place = 0;
        const int leader = __ffs((int)who) - 1;
        if (lane == leader) place = peer_add(peer(&s.taken, 0), __popc(who));
        place = __shfl_sync(0xffffffffu, place, leader) + __popc(who & ((1u << lane) - 1u));
        if (take && place < CAP) peer_st(peer(&s.list[place], 0), key);
    };
    // the first n of the list in descending order (n <= CAP): few by their rank, many by a sort
    auto arrange = [&](int n) {
        if (n > 256) {
            sort_down(s.list, n);
            return;
        }
        const u64 mine = tid < n ? s.list[tid] : 0;
        int rank_of = 0;
        for (int i = 0; i < n; ++i) rank_of += s.list[i] > mine;
        __syncthreads();
        if (tid < n) s.list[rank_of] = mine;
        __syncthreads();
    };

    // The smallest and the largest of the CTA's keys, for every thread.
    auto span_of = [&](u64& kl, u64& kh) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            kl = min(kl, __shfl_xor_sync(0xffffffffu, kl, o));
            kh = max(kh, __shfl_xor_sync(0xffffffffu, kh, o));
        }
        if (lane == 0) {
            s.ends[warp] = kl;
            s.ends[NW + warp] = kh;
        }
        __syncthreads();
        for (int k = 0; k < NW; ++k) {
            kl = min(kl, s.ends[k]);
            kh = max(kh, s.ends[NW + k]);
        }
    };
    bool bracketed = false;   // a border by mass is known to lie between two keys
    u64 bracket[4] = {0, 0, 0, 0};

    if (by_count && top_k <= FEW) {
        // ---- few tokens: the first CTA takes them ----
        spread(COUNT_SPAN);
        for (int i = tid; i < BINS; i += NT) s.count[i] = 0;
        __syncthreads();
        if (2 * top_k <= NT * ranks) {   // the threads' own maxima: top_k of them reach the bound, and so do that many tokens
            if (own_best > -INFINITY) atomicAdd(&s.count[bin_of(own_best)], 1u);
        } else {
            each(-3.402823466e38f, [&](float l, int) {
                if (l > -INFINITY) atomicAdd(&s.count[bin_of(l)], 1u);
            });
        }
        if (ranks > 1) cluster_meet();
        else __syncthreads();
        uint32_t c4[4], total;
        sum_bins(c4);
        uint32_t before = block_scan<uint32_t>(c4[0] + c4[1] + c4[2] + c4[3], s.warp_sum, &total);
        if (tid == 0) s.found[0] = BINS - 1;   // fewer threads with a token than top_k: every token
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (before < (uint32_t)top_k && (uint32_t)top_k <= before + c4[k]) s.found[0] = 4 * tid + k;
            before += c4[k];
        }
        __syncthreads();
        const int bin = (int)s.found[0];
        // (a token of the bin is not below this; the bin itself decides)
        const float low = bin == BINS - 1 || fine == 0.f ? -3.402823466e38f : top - (float)(bin + 2) / fine;
        each(low, [&](float l, int i) { hand_in(l > -INFINITY && bin_of(l) <= bin, place_key(l, lo + i)); });
        if (ranks > 1) cluster_meet();
        else __syncthreads();
        const uint32_t listed = rank == 0 ? (uint32_t)s.taken : peer_ld(peer(&s.taken, 0));
        if (ranks > 1) cluster_meet();   // (the count is read by all before the first CTA goes on)
        if (listed <= CAP) {
            if (rank) return;
            arrange((int)listed);
            const int kept = min(top_k, (int)listed);
            // weights; the tokens before which less than top_p lies; those of min_p or more: each a beginning of the list
            u64* masses = s.list + CAP - FEW;   // [FEW], over what is behind the top_k
            static_assert(2 * FEW <= CAP, "the list's second half");
            constexpr int EACH = FEW / NT;
            u64 sum = 0;
            int left = 0;
            for (int i = tid; i < kept; i += NT) {
                const double z = w.place(logit_of(s.list[i]));
                masses[i] = w.of(z, s.two_to);
                left += z >= floor_z;
            }
            left = block_sum_of(left, s.warp_sum);
            const int i0 = tid * EACH;
            u64 v[EACH], all;
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                v[k] = i0 + k < kept ? masses[i0 + k] : 0;
                sum += v[k];
            }
            u64 lies = block_scan<u64>(sum, s.warp_sum, &all);
            if (by_mass) {
                const double t = (double)top_p * (double)all;
                int in = 0;
#pragma unroll
                for (int k = 0; k < EACH; ++k) {
                    in += i0 + k < kept && (i0 + k == 0 || (double)lies < t);
                    lies += v[k];
                }
                left = min(left, block_sum_of(in, s.warp_sum));
            }
            // what stays, by number
            sum = 0;
#pragma unroll
            for (int k = 0; k < EACH; ++k) sum += i0 + k < left ? v[k] : 0;
            block_scan<u64>(sum, s.warp_sum, &all);
            const u64 target = aim(all);
            if (left <= 256) {   // each token sums the ones of lower numbers for itself
                if (tid < left) {
                    const int number = token_of(s.list[tid]);
                    u64 under = 0;
                    for (int i = 0; i < left; ++i) under += token_of(s.list[i]) < number ? masses[i] : 0;
                    if (under <= target && target < under + masses[tid]) a.out[r] = number;
                }
                return;
            }
            for (int i = tid; i < left; i += NT) s.list[i] = (u64)(uint32_t)s.list[i] << 32 | (uint32_t)i;   // (a key's low word is ~number)
            sort_down(s.list, left);
            sum = 0;
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                v[k] = i0 + k < left ? masses[(uint32_t)s.list[i0 + k]] : 0;
                sum += v[k];
            }
            u64 here = block_scan<u64>(sum, s.warp_sum, &all);
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                if (here <= target && target < here + v[k]) a.out[r] = (int)~(uint32_t)(s.list[i0 + k] >> 32);
                here += v[k];
            }
            return;
        }
    } else if (by_mass && !by_count) {
        // ---- top_p alone ----
        spread(mass_span);
        for (int i = tid; i < BINS; i += NT) s.count[i] = 0;
        __syncthreads();
        // Four tokens side by side and without branches: a weight is a chain of a dozen operations.  (Minus infinity counts
        // for the last bin, whose number is only ever an upper bound, with a weight of 2^-1000: no unit.)
        u64 sum = 0;
        float4 q = own_quad(tid, quads);
        for (int j = tid; j < quads; j += NT) {
            const float4 next = own_quad(j + NT, quads);
            const float l4[4] = {q.x, q.y, q.z, q.w};
            u64 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = w.of(l4[k], s.two_to);
#pragma unroll
            for (int k = 0; k < 4; ++k) atomicAdd(&s.count[bin_of(l4[k])], 1u);
            sum += (v[0] + v[1]) + (v[2] + v[3]);
            q = next;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s.warp_sum[warp] = sum;
        __syncthreads();
        sum = 0;
        for (int k = 0; k < NW; ++k) sum += s.warp_sum[k];
        tell(sum, 0, 0, 0);   // (the counts are there, too)
        sum = 0;
        for (int c = 0; c < ranks; ++c) sum += s.slot[turn][c][0];
        const double whole = (double)sum, t = (double)top_p * whole;
        const u64 target = max(t > 0.0 ? (u64)ceil(t) : 0, 1ull);   // the last token before which less than this lies
        // The bins in which that token can lie: a bin's weights are between those of its edges.  The last bin has no lower edge.
        uint32_t c4[4];
        sum_bins(c4);
        const float octaves = (float)(w.scale * (double)span / (TABLE * BINS));   // of a bin, MASS_SPAN / BINS at most
        const double step = exp2f(-octaves);                                      // of a bin's weights
        double edge = exp2f(-octaves * (4.f * tid)) * ONE;
        double most[4], sum4 = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            most[k] = c4[k] * edge;   // at the upper edge; at the lower one `step` times that
            sum4 += most[k];
            edge *= step;
        }
        if (tid == NT - 1) s.ends[0] = (u64)__double_as_longlong(most[3]);
        double all_bins;
        double here = block_scan_double(sum4, reinterpret_cast<double*>(s.warp_sum), &all_bins);
        const double last_bin = __longlong_as_double((long long)s.ends[0]);
        // (a spread too small to be divided into bins: all that is below the maximum is in the last one, above its edges too)
        const bool told = fine < INFINITY;
        if (tid == 0) s.found[0] = told ? BINS - 1 : 0, s.found[1] = BINS - 1;
        __syncthreads();
        int lo_bin = BINS - 1, hi_bin = BINS - 1;
        // The tokens up to a bin are at least and at most so much by the bins up to it, and by the total less the bins behind
        // it: whichever is less far from its edges (at a top_p of 0.9 the latter, by nine times).
        // margin: of the sums' rounding and of the edges' (fp32: 20 octaves to 2^-24 of them, 2^-19 of a weight); slack: of
        // these sums against the weights in units
        const double margin = 1.0 + 2e-5, slack = whole * 1e-11 + (double)a.vocab;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            here += most[k];
            const double behind = all_bins - here;
            const double high = fmin(here * margin, whole - fmax(behind - last_bin, 0.0) * step / margin) + slack;
            const double least_sum = fmax(here * step / margin, whole - behind * margin) - slack;
            const int b = 4 * tid + k;
            if (high >= (double)target) lo_bin = min(lo_bin, b);
            if (least_sum >= (double)target + 1.0 && b < BINS - 1) hi_bin = min(hi_bin, b);
        }
        if (lo_bin < BINS - 1) atomicMin(&s.found[0], (u64)lo_bin);
        if (hi_bin < BINS - 1 && told) atomicMin(&s.found[1], (u64)hi_bin);
        __syncthreads();
        lo_bin = (int)s.found[0];
        hi_bin = (int)s.found[1];
        // tokens above those bins stay: their weights, and those of min_p or more by pieces of the row; the bins' own tokens
        // go to the first CTA.  A piece is a run of quads to a warp.
        const int piece = ceil_div(quads, NW), q0 = min(quads, warp * piece), q1 = min(quads, q0 + piece);
        const float low = hi_bin == BINS - 1 || fine == 0.f ? -3.402823466e38f : top - (float)(hi_bin + 2) / fine;
        u64 above = 0, stay = 0, kl = ~0ull, kh = 0;   // kl, kh: of the bins' tokens
        float4 ahead = own_quad(q0 + lane, q1);
        for (int j = q0 + lane; j < ((q1 - q0 + 31) & ~31) + q0; j += 32) {
            const float4 q = ahead;
            ahead = own_quad(j + 32, q1);
            if (!__any_sync(0xffffffffu, fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)) >= low)) continue;
            const float l4[4] = {q.x, q.y, q.z, q.w};
            bool take[4], any = false;
            unsigned over = 0;   // tokens above the bins
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int b = bin_of(l4[k]);
                const bool there = l4[k] > -INFINITY;
                take[k] = there && b >= lo_bin && b <= hi_bin;
                any |= take[k];
                over |= (unsigned)(there && b < lo_bin) << k;
            }
            while (__any_sync(0xffffffffu, over)) {   // few of a warp's 128, as a rule: each lane's next one
                const int k = __ffs((int)over) - 1;
                const float l = k == 0 ? q.x : k == 1 ? q.y : k == 2 ? q.z : q.w;
                const double z = w.place(l);
                const u64 v = over ? w.of(z, s.two_to) : 0;
                above += v;
                if (z >= floor_z) stay += v;
                over &= over - 1;
            }
            if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const u64 key = place_key(l4[k], lo + 4 * j + k - off);
                if (take[k]) kl = min(kl, key), kh = max(kh, key);
                hand_in(take[k], key);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            above += __shfl_xor_sync(0xffffffffu, above, o);
            stay += __shfl_xor_sync(0xffffffffu, stay, o);
        }
        if (lane == 0) {
            s.warp_sum[warp] = above;
            peer_st(peer(&s.pieces[rank * NW + warp], 0), stay);
        }
        __syncthreads();
        above = 0;
        for (int k = 0; k < NW; ++k) above += s.warp_sum[k];
        span_of(kl, kh);
        tell(above, kl, kh, 0);
        const uint32_t listed = rank == 0 ? (uint32_t)s.taken : peer_ld(peer(&s.taken, 0));
        u64 before = 0;
        for (int c = 0; c < ranks; ++c) {
            before += s.slot[turn][c][0];
            kl = min(kl, s.slot[turn][c][1]);
            kh = max(kh, s.slot[turn][c][2]);
        }
        bracketed = true;
        bracket[0] = target, bracket[1] = kl, bracket[2] = kh, bracket[3] = before;
        if (listed <= CAP) {   // all CTAs alike
            if (ranks > 1) cluster_meet();   // (the number is read by all before the first CTA goes on)
            if (rank) return;                // the rest is too little for all: other rows have the room
            arrange((int)listed);
            // the last token of the list before which less than `target` lies, and the tokens up to it that stay
            constexpr int EACH = CAP / NT;
            double z[EACH];
            u64 v[EACH], mine = 0, total;
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                const int i = tid * EACH + k;
                z[k] = i < (int)listed ? w.place(logit_of(s.list[i])) : -INFINITY;
                v[k] = w.of(z[k], s.two_to);
                mine += v[k];
            }
            u64 lies = before + block_scan<u64>(mine, s.warp_sum, &total);
            uint32_t last = 0;
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                const int i = tid * EACH + k;
                if (i < (int)listed && lies < target) {
                    last = i + 1;
                    if (z[k] >= floor_z) {
                        const int number = token_of(s.list[i]), c = number / a.share;
                        const int o = (int)((reinterpret_cast<uintptr_t>(row + (long long)c * a.share) & 15) / sizeof(T));
                        const int in = number - c * a.share + o, all_in = min(a.vocab - c * a.share, a.share) + o;
                        atomicAdd(&s.pieces[c * NW + in / 4 / ceil_div((all_in + 3) / 4, NW)], v[k]);
                    }
                }
                lies += v[k];
            }
            last = __reduce_max_sync(0xffffffffu, last);
            __syncthreads();
            if (lane == 0) s.warp_sum[warp] = last;
            __syncthreads();
            u64 most_at = 1;
            for (int k = 0; k < NW; ++k) most_at = max(most_at, s.warp_sum[k]);
            __syncthreads();   // (read by all before the next scan writes there)
            // the piece in which the token lies, and what its tokens' sum has to exceed
            const u64 bar = listed ? s.list[most_at - 1] : 0;
            const u64 here = tid < ranks * NW ? s.pieces[tid] : 0;
            u64 left_over;
            if (tid == 0) s.found[0] = s.found[1] = 0;
            const u64 passed = block_scan<u64>(here, s.warp_sum, &left_over);
            const u64 goal = aim(left_over);
            if (passed <= goal && goal < passed + here) s.found[0] = (u64)tid, s.found[1] = goal - passed;
            __syncthreads();
            const unsigned which = (unsigned)s.found[0];
            const int c = (int)(which / NW);
            const u64 rest = s.found[1];
            const T* xc = row + (long long)c * a.share;   // of that CTA's share
            const int oc = (int)((reinterpret_cast<uintptr_t>(xc) & 15) / sizeof(T)), nc = min(a.vocab - c * a.share, a.share);
            const int qc = (oc + nc + 3) / 4, pc = ceil_div(qc, NW);
            const int p0 = min(qc, (int)(which % NW) * pc), p1 = min(qc, p0 + pc);
            const int per = ceil_div(4 * (p1 - p0), NT), e0 = min(4 * p1, 4 * p0 + tid * per), e1 = min(4 * p1, e0 + per);
            auto weight_at = [&](int e) -> u64 {   // of place e among the quads
                const int i = e - oc;
                if (i < 0 || i >= nc) return 0;
                const float l = clean(load_one(xc + i));
                if (l == -INFINITY || place_key(l, c * a.share + i) < bar) return 0;
                const double z = w.place(l);
                return z >= floor_z ? w.of(z, s.two_to) : 0;
            };
            u64 sum_here = 0, all;
            for (int e = e0; e < e1; ++e) sum_here += weight_at(e);
            u64 at_e = block_scan<u64>(sum_here, s.warp_sum, &all);
            if (at_e <= rest && rest < at_e + sum_here)
                for (int e = e0; e < e1; ++e) {
                    at_e += weight_at(e);
                    if (rest < at_e) {
                        a.out[r] = c * a.share + e - oc;
                        break;
                    }
                }
            return;
        }
    }

    // ---- the general form ----
    u64 bar = 0;   // tokens whose key is below this are out
    auto low_of = [&](u64 key) { return key ? logit_of(key) : -3.402823466e38f; };
    // The key of the last token that stays: by count the want-th, by mass the last one before which less than `want` lies
    // (0: top_p of the sum).  The range of keys in which it is looked for is cut into bins, from the top down, until a bin's
    // tokens can be sorted; `before` of the order (tokens or weight) has passed when the range begins.  With `first`, the
    // range is everything, and the bins are of equal width in the logit.
    auto border = [&](bool mass, u64 want, bool first_level, u64 lo_key, u64 hi_key, u64 before) -> u64 {
        if (first_level) spread(mass ? mass_span : COUNT_SPAN);
        u64 target = want, count = 0;
        int bin = 0, shift = 0;
        auto cut = [&]() { shift = max(0, 64 - __clzll((long long)(hi_key - lo_key)) - 11); };   // 2048 bins
        if (!first_level) cut();
        while (true) {
            for (int i = tid; i < BINS; i += NT) s.count[i] = s.low[i] = s.high[i] = 0;
            __syncthreads();
            const u64 from = max(bar, lo_key);
            each(low_of(from), [&](float l, int i) {
                const u64 key = place_key(l, lo + i);
                if (l == -INFINITY || key < from || key > hi_key) return;
                const int b = first_level ? bin_of(l) : (int)((hi_key - key) >> shift);
                atomicAdd(&s.count[b], 1u);
                if (mass) {
                    const u64 v = w.of(l, s.two_to);
                    if (v) {
                        const uint32_t lo32 = (uint32_t)v, old = atomicAdd(&s.low[b], lo32);
                        const uint32_t hi32 = (uint32_t)(v >> 32) + (old + lo32 < old ? 1u : 0u);
                        if (hi32) atomicAdd(&s.high[b], hi32);
                    }
                }
            });
            if (ranks > 1) cluster_meet();
            else __syncthreads();
            // four bins to a thread, over all CTAs
            uint32_t c4[4];
            sum_bins(c4);
            u64 m4[4] = {c4[0], c4[1], c4[2], c4[3]};
            if (mass) {
                m4[0] = m4[1] = m4[2] = m4[3] = 0;
                for (int c = 0; c < ranks; ++c) {
                    const uint4 l = peer_ld4(peer(&s.low[4 * tid], c)), h = peer_ld4(peer(&s.high[4 * tid], c));
                    m4[0] += (u64)h.x << 32 | l.x, m4[1] += (u64)h.y << 32 | l.y;
                    m4[2] += (u64)h.z << 32 | l.z, m4[3] += (u64)h.w << 32 | l.w;
                }
            }
            u64 total;
            u64 at_bin = before + block_scan<u64>(m4[0] + m4[1] + m4[2] + m4[3], s.warp_sum, &total);
            if (!mass && before + total < target) {   // fewer tokens than that: all stay
                if (ranks > 1) cluster_meet();        // (the counts are read by all before they are cleared again)
                else __syncthreads();
                return bar;
            }
            if (mass && !target) {
                const double t = (double)top_p * (double)total;
                target = max(t > 0.0 ? (u64)ceil(t) : 0, 1ull);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (at_bin < target && target <= at_bin + m4[k]) {
                    s.found[0] = 4 * tid + k;
                    s.found[1] = at_bin;
                    s.found[2] = c4[k];
                }
                at_bin += m4[k];
            }
            __syncthreads();
            bin = (int)s.found[0];
            before = s.found[1];
            count = s.found[2];
            __syncthreads();
            if (!first_level) {
                hi_key -= (u64)bin << shift;
                lo_key = max(lo_key, hi_key - ((1ull << shift) - 1));
            }
            if (count <= CAP) break;
            // too many: the keys of the bin, cut again
            if (first_level) {
                u64 kl = ~0ull, kh = 0;
                each(low_of(bar), [&](float l, int i) {
                    const u64 key = place_key(l, lo + i);
                    if (l == -INFINITY || key < bar || bin_of(l) != bin) return;
                    kl = min(kl, key);
                    kh = max(kh, key);
                });
                span_of(kl, kh);
                tell(kl, kh, 0, 0);
                lo_key = ~0ull;
                hi_key = 0;
                for (int c = 0; c < ranks; ++c) {
                    lo_key = min(lo_key, s.slot[turn][c][0]);
                    hi_key = max(hi_key, s.slot[turn][c][1]);
                }
                first_level = false;
            } else if (ranks > 1) {
                cluster_meet();   // the counts are read before they are cleared
            }
            cut();
        }
        // the bin's tokens, in every CTA's list
        uint32_t base = 0;
        for (int c = 0; c < rank; ++c) base += peer_ld(peer(&s.count[bin], c));
        if (tid == 0) s.taken = 0;
        if (ranks > 1) cluster_meet();   // the sums are read by all
        else __syncthreads();
        const u64 from = max(bar, lo_key);
        each(low_of(from), [&](float l, int i) {
            const u64 key = place_key(l, lo + i);
            if (l == -INFINITY || key < from || key > hi_key || (first_level && bin_of(l) != bin)) return;
            const uint32_t place = base + atomicAdd(&s.taken, 1);
            for (int c = 0; c < ranks; ++c) peer_st(peer(&s.list[place], c), key);
        });
        if (ranks > 1) cluster_meet();
        else __syncthreads();
        arrange((int)count);
        if (!mass) {
            const u64 key = s.list[target - before - 1];
            __syncthreads();
            return key;
        }
        // the last of the list before which less than `target` lies
        constexpr int EACH = CAP / NT;
        u64 v[EACH], sum = 0, total;
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int i = tid * EACH + k;
            v[k] = i < (int)count ? w.of(logit_of(s.list[i]), s.two_to) : 0;
            sum += v[k];
        }
        u64 lies = before + block_scan<u64>(sum, s.warp_sum, &total);
        uint32_t last = 0;
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int i = tid * EACH + k;
            if (i < (int)count && lies < target) last = i + 1;
            lies += v[k];
        }
        last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) s.warp_sum[warp] = last;
        __syncthreads();
        u64 most = 1;
        for (int k = 0; k < NW; ++k) most = max(most, s.warp_sum[k]);
        const u64 key = s.list[most - 1];
        __syncthreads();
        return key;
    };
    if (bracketed) {
        bar = border(true, bracket[0], false, bracket[1], bracket[2], bracket[3]);
    } else {
        if (by_count) bar = border(false, (u64)top_k, true, 0, ~0ull, 0);
        if (by_mass) bar = border(true, 0, true, 0, ~0ull, 0);
    }

    // the sums of what stays, in the order of the tokens: a run of the share to a warp
    const float low = low_of(bar);
    auto weight_at = [&](int e) -> u64 {   // of place e
        const int i = e - off;
        if (i < 0 || i >= n) return 0;
        const float l = at(i);
        if (!(l >= low) || place_key(l, lo + i) < bar) return 0;
        const double z = w.place(l);
        return z >= floor_z ? w.of(z, s.two_to) : 0;
    };
    const int piece = ceil_div(quads, NW), q0 = min(quads, warp * piece), q1 = min(quads, q0 + piece);
    u64 sum = 0;
    for (int j = q0 + lane; j < q1; j += 32) {
        const float4 q = quad(j);
        if (!(fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)) >= low)) continue;
        const float l4[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (!(l4[k] >= low) || place_key(l4[k], lo + 4 * j + k - off) < bar) continue;
            const double z = w.place(l4[k]);
            if (z >= floor_z) sum += w.of(z, s.two_to);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s.warp_sum[warp] = sum;
    __syncthreads();
    u64 mine = 0;
    for (int k = 0; k < NW; ++k) mine += s.warp_sum[k];
    tell(mine, 0, 0, 0);
    u64 total = 0, begin = 0;
    for (int c = 0; c < ranks; ++c) {
        if (c == rank) begin = total;
        total += s.slot[turn][c][0];
    }
    const u64 target = aim(total);
    if (target < begin || target - begin >= mine) return;
    u64 passed = begin;
    int k = 0;
    for (; k < NW - 1 && target >= passed + s.warp_sum[k]; ++k) passed += s.warp_sum[k];
    __syncthreads();
    // the run, over all threads
    const int p0 = 4 * min(quads, k * piece), p1 = 4 * min(quads, (k + 1) * piece), per = ceil_div(p1 - p0, NT);
    const int j0 = min(p1, p0 + tid * per), j1 = min(p1, j0 + per);
    sum = 0;
    for (int e = j0; e < j1; ++e) sum += weight_at(e);
    u64 all;
    u64 here = passed + block_scan<u64>(sum, s.warp_sum, &all);
    if (here <= target && target < here + sum)
        for (int e = j0; e < j1; ++e) {
            here += weight_at(e);
            if (target < here) {
                a.out[r] = lo + e - off;
                break;
            }
        }
}

size_t smem_of(int share, bool near) {
    return ((sizeof(Shared) + 15) & ~(size_t)15) + (near ? (size_t)share * 4 + 64 : 0);
}

template <typename T>
int run(Args a, cudaStream_t st) {
    // As many CTAs to a row as leave each 4096 tokens or more.  Two of a row of 152k fit an SM; with one CTA to a row, and
    // passes that read it from L2, 256 rows took 466 us and not 390 as the kernel was then (64 rows: 129 and 92).
    unsigned ranks = 1;
    while (ranks < MAX_RANKS && a.vocab > 4096 * (int)ranks) ranks *= 2;
    a.share = (ceil_div(a.vocab, (int)ranks) + 7) & ~7;
    const bool near = smem_of(a.share, true) <= 220 * 1024;
    const size_t smem = smem_of(a.share, near);
    static SmemLimit limits[2];
    const auto kernel = near ? sample_kernel<T, true> : sample_kernel<T, false>;
    cudaError_t e = allow_smem(kernel, smem, limits[near]);
    if (e == cudaSuccess) e = launch_cluster(kernel, (unsigned)a.n * ranks, ranks, dim3(NT), smem, st, a);
    return e == cudaSuccess ? MQ_OK : note_cuda(e, "sample");
}

}  // namespace sampling
}  // namespace mq

extern "C" int mq_sample(const mq_sample_params* p, cudaStream_t st) {
    if (!p || p->n < 0 || p->vocab < 1 || p->vocab > mq::sampling::MAX_VOCAB || p->n > (1 << 24)) return MQ_ERR_INVALID_ARGUMENT;
    if (!p->n) return MQ_OK;
    const size_t size = p->dtype == MQ_FP32 ? 4 : 2;
    if (!p->logits || !p->u || !p->tokens || (reinterpret_cast<uintptr_t>(p->logits) % size) ||
        (p->dtype != MQ_FP32 && p->dtype != MQ_BF16 && p->dtype != MQ_FP16))
        return MQ_ERR_INVALID_ARGUMENT;
    mq::sampling::Args a = {};
    a.logits = p->logits;
    a.row = p->row_stride;
    a.n = p->n;
    a.vocab = p->vocab;
    a.u = p->u;
    a.temperature = p->temperatures;
    a.top_k = p->top_ks;
    a.top_p = p->top_ps;
    a.min_p = p->min_ps;
    a.temperature_v = p->temperature;
    a.top_k_v = p->top_k;
    a.top_p_v = p->top_p;
    a.min_p_v = p->min_p;
    a.out = p->tokens;
    return p->dtype == MQ_FP32   ? mq::sampling::run<float>(a, st)
           : p->dtype == MQ_BF16 ? mq::sampling::run<__nv_bfloat16>(a, st)
                                 : mq::sampling::run<__half>(a, st);
}
