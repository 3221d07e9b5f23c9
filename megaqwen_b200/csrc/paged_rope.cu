// Rotary positions fused with the write of K and V into the paged cache, and
// the pages' score index.
//
// Memory-bound: each token's q, k and v are read once and written once,
// (Hq + 2 Hkv) D elements each way; the cos/sin row of a token is shared by its
// heads and comes from L1.  32008 tokens of 16 + 8 + 8 heads x 128, 528 MB: 92 us,
// 5.7 TB/s, 0.88 of the copy rate (with the index 114 us: its 65 MB of keys are
// read again).
#include <algorithm>

#include "paged_common.cuh"

namespace mq {
namespace paged {

constexpr int ROPE_THREADS = 128;

struct RopeArgs {
    const uint16_t* q;
    uint16_t* q_out;
    const uint16_t* k;
    const uint16_t* v;
    long long q_tok, q_head, o_tok, o_head, k_tok, k_head, v_tok, v_head;
    const int* positions;
    const int* places;   // null: the positions
    const int* slots;
    const float* cos_t;
    const float* sin_t;
    long long cos_row, sin_row;
    int max_pos, hq, hkv, rot, inverse;
    uint16_t* kp;     // pages, at the layer
    uint16_t* vp;
    long long kp_page, kp_head, vp_page, vp_head;
    const int* table;
    long long table_row;
    int slots_n, cols, pages, page, shift;   // page = 1 << shift
    int* status;
};

// The products and sums are rounded one by one (no FMA), so the result is that
// of the plain formula in fp32 and not of the compiler's contraction.
__device__ __forceinline__ void turn(float& x0, float& x1, float c, float s) {
    const float a = x0, b = x1;
    x0 = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    x1 = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}

// Where a token goes.  page -1: nowhere (no cache, or a wrong place).
struct Place {
    int pos, page, row;
    bool ok;   // the position is inside the tables
};
__device__ __forceinline__ Place place_of(const RopeArgs& a, int pos, int at, int slot, bool report) {
    Place p;
    p.pos = pos;
    p.page = -1;
    p.row = 0;
    p.ok = pos >= 0 && pos < a.max_pos;
    if (!p.ok) {
        if (report) note_status(a.status, MQ_ERR_BAD_POSITION);
    } else if (a.kp) {
        const int c = at >> a.shift;
        if (slot < 0 || slot >= a.slots_n) {
            if (report) note_status(a.status, MQ_ERR_BAD_SLOT);
        } else if (at < 0 || c >= a.cols) {
            if (report) note_status(a.status, MQ_ERR_BAD_POSITION);
        } else {
            const int g = __ldg(a.table + slot * a.table_row + c);
            if (g >= 0 && g < a.pages) {
                p.page = g;
                p.row = at & (a.page - 1);
            } else if (report) {
                note_status(a.status, MQ_ERR_BAD_PAGE);
            }
        }
    }
    return p;
}

// Head h of a token: q heads first, then k, then v.
__device__ __forceinline__ const uint16_t* src_of(const RopeArgs& a, int t, int h) {
    if (h < a.hq) return a.q + t * a.q_tok + h * a.q_head;
    h -= a.hq;
    return h < a.hkv ? a.k + t * a.k_tok + h * a.k_head : a.v + t * a.v_tok + (h - a.hkv) * a.v_head;
}
// Where it is written, or null.
__device__ __forceinline__ uint16_t* dst_of(const RopeArgs& a, int t, int h, int D, const Place& p) {
    if (h < a.hq) return a.q_out + t * a.o_tok + h * a.o_head;
    if (p.page < 0) return nullptr;
    h -= a.hq;
    return h < a.hkv ? a.kp + p.page * a.kp_page + h * a.kp_head + p.row * D
                     : a.vp + p.page * a.vp_page + (h - a.hkv) * a.vp_head + p.row * D;
}

// Vector path: rotary_dim a multiple of 16, every address a multiple of 16
// bytes.  A unit is two pieces of 8 channels of a head, chosen so that a piece's
// neighbour lane has the neighbouring piece: for the half layout the 8 pairs
// (8u + i, 8u + i + R / 2), or two pieces past R; interleaved, pieces u and
// D / 16 + u, each four pairs or past R.
//
// Each CTA walks over tokens, two heads of a thread at a time.  The next step's
// reads are issued before the present one's writes, and a token's position is
// read a step before its place in the table and its cos/sin: in a CTA of its own
// per token these reads come one after another and leave the memory idle between
// (95 us for 530 MB).
template <typename T, int D, bool INTER, bool PLACED>   // PLACED: K and V have places of their own (117.7 us in one kernel, not 114.3)
__global__ void __launch_bounds__(ROPE_THREADS, 8) rope_kernel(const RopeArgs a, int n) {
    constexpr int UNITS = D / 16, LANES = ROPE_THREADS / UNITS;
    pdl_wait();
    pdl_trigger();
    const int u = threadIdx.x % UNITS, lane_h = threadIdx.x / UNITS;
    const int heads = a.hq + (a.kp ? 2 * a.hkv : 0);
    // first channels of the two pieces, and whether they are turned
    const int pairs = a.rot / 16;   // half layout: units that turn
    const int r0 = INTER || u < pairs ? 8 * u : a.rot + 8 * (u - pairs);
    const int r1 = INTER ? D / 2 + 8 * u : u < pairs ? r0 + a.rot / 2 : r0 + (D - a.rot) / 2;
    const bool turn0 = r0 < a.rot, turn1 = INTER ? r1 < a.rot : turn0;
    uint4 x[2], y[2];   // what the step in hand turns; refilled for the next one as it is written
    auto read = [&](int t, int h, int i) {
        if (h + i * LANES >= heads) return;
        const uint16_t* src = src_of(a, t, h + i * LANES);
        x[i] = __ldcs(reinterpret_cast<const uint4*>(src + r0));
        y[i] = __ldcs(reinterpret_cast<const uint4*>(src + r1));
    };
    int t = blockIdx.x, h = lane_h;
    if (t >= n) return;
    int pos = __ldg(a.positions + t), slot = a.kp ? __ldg(a.slots + t) : 0, at = PLACED ? __ldg(a.places + t) : 0;
    read(t, h, 0);
    read(t, h, 1);
    Place p;
    float cs[8], sn[8];
    while (t < n) {
        if (h == lane_h) {   // a new token
            p = place_of(a, pos, PLACED ? at : pos, slot, threadIdx.x == 0);
            if (turn0 && p.ok) {
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    if (i && !turn1) break;   // (half layout: both or none)
                    const int pair = INTER ? (i ? r1 : r0) / 2 : r0 + i;
                    const float4 c = __ldg(reinterpret_cast<const float4*>(a.cos_t + pos * a.cos_row + pair));
                    const float4 s = __ldg(reinterpret_cast<const float4*>(a.sin_t + pos * a.sin_row + pair));
                    cs[i] = c.x; cs[i + 1] = c.y; cs[i + 2] = c.z; cs[i + 3] = c.w;
                    sn[i] = s.x; sn[i + 1] = s.y; sn[i + 2] = s.z; sn[i + 3] = s.w;
                }
                if (a.inverse) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) sn[i] = -sn[i];
                }
            }
            if (t + (int)gridDim.x < n) {
                pos = __ldg(a.positions + t + gridDim.x);
                if (a.kp) slot = __ldg(a.slots + t + gridDim.x);
                if (PLACED) at = __ldg(a.places + t + gridDim.x);
            }
        }
        int t1 = t, h1 = h + 2 * LANES;   // the next step
        if (h1 >= heads) {
            t1 += gridDim.x;
            h1 = lane_h;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint4 v = x[i], w = y[i];
            const int hh = h + i * LANES;
            if (t1 < n) read(t1, h1, i);
            if (hh >= heads) continue;
            uint16_t* dst = dst_of(a, t, hh, D, p);
            if (!dst) continue;
            if (!p.ok) {
                v = w = make_uint4(0, 0, 0, 0);   // a position outside the tables has no rotation
            } else if (turn0 && hh < a.hq + a.hkv) {
                uint32_t* xv = reinterpret_cast<uint32_t*>(&v);
                uint32_t* yv = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float2 e = Elem<T>::up2(xv[k]), f = Elem<T>::up2(yv[k]);
                    if (INTER) {   // pairs are neighbours
                        turn(e.x, e.y, cs[k], sn[k]);
                        if (turn1) turn(f.x, f.y, cs[4 + k], sn[4 + k]);
                    } else {
                        turn(e.x, f.x, cs[2 * k], sn[2 * k]);
                        turn(e.y, f.y, cs[2 * k + 1], sn[2 * k + 1]);
                    }
                    xv[k] = Elem<T>::pack(e.x, e.y);
                    if (!INTER || turn1) yv[k] = Elem<T>::pack(f.x, f.y);
                }
            }
            // everything but K streams through L2 (read and written once here), so that the index
            // kernel finds the keys there (65 MB of them among 530 MB)
            if (hh >= a.hq && hh < a.hq + a.hkv) {
                *reinterpret_cast<uint4*>(dst + r0) = v;
                *reinterpret_cast<uint4*>(dst + r1) = w;
            } else {
                __stcs(reinterpret_cast<uint4*>(dst + r0), v);
                __stcs(reinterpret_cast<uint4*>(dst + r1), w);
            }
        }
        t = t1;
        h = h1;
    }
}

// Any even rotary_dim and any alignment: a thread per pair of channels.
template <typename T>
__global__ void __launch_bounds__(ROPE_THREADS) rope_any_kernel(const RopeArgs a, int D, int inter) {
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x, half = a.rot / 2;
    const int pos = __ldg(a.positions + t);
    const Place p = place_of(a, pos, a.places ? __ldg(a.places + t) : pos, a.kp ? __ldg(a.slots + t) : 0, threadIdx.x == 0);
    const int heads = a.hq + (a.kp ? 2 * a.hkv : 0);
    for (int e = threadIdx.x; e < heads * (D / 2); e += ROPE_THREADS) {
        const int h = e / (D / 2), i = e - h * (D / 2);
        const uint16_t* src = src_of(a, t, h);
        uint16_t* dst = dst_of(a, t, h, D, p);
        if (!dst) continue;
        const bool in = i < half;
        const int c0 = in && !inter ? i : 2 * i, c1 = in && !inter ? i + half : 2 * i + 1;
        uint16_t x = src[c0], y = src[c1];
        if (!p.ok) x = y = 0;
        if (h < a.hq + a.hkv && in && p.ok) {
            float f = Elem<T>::up(x), g = Elem<T>::up(y);
            const float c = a.cos_t[p.pos * a.cos_row + i], s = a.sin_t[p.pos * a.sin_row + i];
            turn(f, g, c, a.inverse ? -s : s);
            x = Elem<T>::down(f);
            y = Elem<T>::down(g);
        }
        dst[c0] = x;
        dst[c1] = y;
    }
}

// ---- the index of full pages ------------------------------------------------------------
// CTA (chunk of 512 tokens, kv head): the tokens of the chunk that are the last
// row of their page are dealt to its warps; a warp takes the bounds of one
// page's keys (read from L2, where the kernel before left them, eight rows of
// 16 bytes a lane in flight).  Bounds are exact (no arithmetic on the keys), so
// the record does not depend on the order of the rows.
constexpr int INDEX_THREADS = 256, INDEX_TOKENS = 512;

template <typename T, int D>
__global__ void __launch_bounds__(INDEX_THREADS) index_kernel(const RopeArgs a, int n, signed char* __restrict__ index,
                                                              long long i_page, long long i_head) {
    constexpr int PIECES = D / 8, ROWS = 32 / PIECES;   // 8 channels a lane, ROWS rows side by side
    __shared__ int list[INDEX_TOKENS];
    __shared__ int count;
    pdl_wait();
    pdl_trigger();
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const int h = blockIdx.y;
#pragma unroll
    for (int i = 0; i < INDEX_TOKENS; i += INDEX_THREADS) {
        const int t = blockIdx.x * INDEX_TOKENS + i + threadIdx.x;
        if (t >= n) break;
        const int pos = __ldg(a.positions + t), slot = __ldg(a.slots + t);
        const int at = a.places ? __ldg(a.places + t) : pos;
        if ((at & (a.page - 1)) == a.page - 1) {
            const Place p = place_of(a, pos, at, slot, false);
            if (p.page >= 0) list[atomicAdd(&count, 1)] = p.page;
        }
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, piece = lane % PIECES;
    for (int e = threadIdx.x >> 5; e < count; e += INDEX_THREADS / 32) {
        const uint16_t* k = a.kp + list[e] * a.kp_page + h * a.kp_head + (lane / PIECES) * D + piece * 8;
        float hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            hi[i] = -INFINITY;
            lo[i] = INFINITY;
        }
        for (int r = 0; r < a.page; r += 8 * ROWS) {   // page >= 16: with two rows side by side one batch, or more
            uint4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = r + i * ROWS;   // past the page (16 rows, four side by side): the first rows again
                x[i] = *reinterpret_cast<const uint4*>(k + (row < a.page ? row : 0) * D);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float2 f = Elem<T>::up2(w[c]);
                    hi[2 * c] = fmaxf(hi[2 * c], f.x);
                    lo[2 * c] = fminf(lo[2 * c], f.x);
                    hi[2 * c + 1] = fmaxf(hi[2 * c + 1], f.y);
                    lo[2 * c + 1] = fminf(lo[2 * c + 1], f.y);
                }
            }
        }
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int o = PIECES; o < 32; o <<= 1) {
                hi[i] = fmaxf(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
                lo[i] = fminf(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
            }
            // infinite keys count as the type's largest, and a channel of nothing but NaN as zero
            if (!(hi[i] >= lo[i])) hi[i] = lo[i] = 0.f;
            hi[i] = fminf(fmaxf(hi[i], -Elem<T>::MAX), Elem<T>::MAX);
            lo[i] = fminf(fmaxf(lo[i], -Elem<T>::MAX), Elem<T>::MAX);
            m = fmaxf(m, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
        }
#pragma unroll
        for (int o = 1; o < PIECES; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const int ex = m > 0.f ? min(max(ilogbf(m) - 6, -60), 40) : 0;
        const float unit = __int_as_float((127 - ex) << 23);   // 2^-ex
        signed char* rec = index + list[e] * i_page + h * i_head;
        if (lane < PIECES) {
            auto whole = [&](const float* v) {
                uint32_t w[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    w[i >> 2] |= (uint32_t)((int)fminf(fmaxf(rintf(v[i] * unit), -127.f), 127.f) & 255) << (8 * (i & 3));
                return make_uint2(w[0], w[1]);
            };
            *reinterpret_cast<uint2*>(rec + piece * 8) = whole(hi);
            *reinterpret_cast<uint2*>(rec + D + piece * 8) = whole(lo);
        } else if (lane == PIECES) {
            *reinterpret_cast<uint4*>(rec + 2 * D) = make_uint4((uint32_t)(ex & 255), 0, 0, 0);
        }
    }
}

template <typename T>
cudaError_t index_layer(const mq_paged_pool* p, const RopeArgs& a, int layer, int n, cudaStream_t st) {
    signed char* ix = p->index + layer * p->i_layer;
    const dim3 chunks(ceil_div(n, INDEX_TOKENS), p->num_kv_heads);
    return p->head_dim == 128 ? launch(index_kernel<T, 128>, chunks, dim3(INDEX_THREADS), 0, st, a, n, ix, p->i_page, p->i_head)
                              : launch(index_kernel<T, 64>, chunks, dim3(INDEX_THREADS), 0, st, a, n, ix, p->i_page, p->i_head);
}

template <typename T>
int run_rope(const mq_rope_params* p, const RopeArgs& a, bool vec, cudaStream_t st) {
    const int D = p->head_dim;
    const dim3 grid(std::min(p->n, 8 * sm_count()));
    cudaError_t e;
    auto go = [&](auto kernel) { return launch(kernel, grid, dim3(ROPE_THREADS), 0, st, a, p->n); };
    if (!vec)
        e = launch(rope_any_kernel<T>, dim3(p->n), dim3(ROPE_THREADS), 0, st, a, D, p->interleaved);
    else if (a.places && D == 128)
        e = p->interleaved ? go(rope_kernel<T, 128, true, true>) : go(rope_kernel<T, 128, false, true>);
    else if (a.places)
        e = p->interleaved ? go(rope_kernel<T, 64, true, true>) : go(rope_kernel<T, 64, false, true>);
    else if (D == 128)
        e = p->interleaved ? go(rope_kernel<T, 128, true, false>) : go(rope_kernel<T, 128, false, false>);
    else
        e = p->interleaved ? go(rope_kernel<T, 64, true, false>) : go(rope_kernel<T, 64, false, false>);
    if (e != cudaSuccess) return note_cuda(e, "rope");
    if (!p->pool || !p->pool->index) return MQ_OK;
    e = index_layer<T>(p->pool, a, p->layer, p->n, st);
    return e == cudaSuccess ? MQ_OK : note_cuda(e, "page index");
}

int reindex(const mq_paged_pool* p, const int* table, long long table_row, int num_slots, int cols, const int* positions,
            const int* slots, int n, cudaStream_t st) {
    RopeArgs a = {};
    a.positions = positions;
    a.slots = slots;
    a.max_pos = 0x7fffffff;
    a.kp_page = p->k_page;
    a.kp_head = p->k_head;
    a.table = table;
    a.table_row = table_row;
    a.slots_n = num_slots;
    a.cols = cols;
    a.pages = p->num_pages;
    a.page = p->page_size;
    a.shift = __builtin_ctz((unsigned)p->page_size);
    for (int l = 0; l < p->num_layers; ++l) {
        a.kp = (uint16_t*)p->k + l * p->k_layer;
        const cudaError_t e = p->dtype == MQ_BF16 ? index_layer<__nv_bfloat16>(p, a, l, n, st) : index_layer<__half>(p, a, l, n, st);
        if (e != cudaSuccess) return note_cuda(e, "page index");
    }
    return MQ_OK;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace paged
}  // namespace mq

using namespace mq::paged;

extern "C" int mq_rope(const mq_rope_params* p, cudaStream_t st) {
    if (!p || p->n < 0 || (p->head_dim != 64 && p->head_dim != 128) || p->rotary_dim < 0 || p->rotary_dim > p->head_dim ||
        p->rotary_dim % 2 || p->num_q_heads < 0 || p->max_pos < 1 || (p->dtype != MQ_BF16 && p->dtype != MQ_FP16) ||
        (p->num_q_heads && p->n && (!p->q || !p->q_out)) || (p->n && !p->positions) ||
        (p->rotary_dim && (!p->cos_table || !p->sin_table)) || (!p->pool && !p->num_q_heads))
        return MQ_ERR_INVALID_ARGUMENT;
    if (p->pool && (!pool_ok(p->pool) || p->pool->dtype != p->dtype || p->pool->head_dim != p->head_dim || p->layer < 0 ||
                    p->layer >= p->pool->num_layers || p->table_cols < 1 || p->num_slots < 1 || !p->table ||
                    (p->n && (!p->k || !p->v || !p->slots))))
        return MQ_ERR_INVALID_ARGUMENT;
    if (!p->n) return MQ_OK;
    RopeArgs a = {};
    a.q = (const uint16_t*)p->q;
    a.q_out = (uint16_t*)p->q_out;
    a.q_tok = p->q_token; a.q_head = p->q_head;
    a.o_tok = p->out_token; a.o_head = p->out_head;
    a.positions = p->positions;
    a.cos_t = p->cos_table;
    a.sin_t = p->sin_table;
    a.cos_row = p->cos_row;
    a.sin_row = p->sin_row;
    a.max_pos = p->max_pos;
    a.hq = p->num_q_heads;
    a.rot = p->rotary_dim;
    a.inverse = p->inverse;
    a.status = p->status;
    long long odd = (p->q_token | p->q_head | p->out_token | p->out_head) % 8;
    bool vec = p->rotary_dim % 16 == 0 && al16(p->q) && al16(p->q_out) && al16(p->cos_table) && al16(p->sin_table) &&
               p->cos_row % 4 == 0 && p->sin_row % 4 == 0;
    if (p->pool) {
        const mq_paged_pool& o = *p->pool;
        a.k = (const uint16_t*)p->k;
        a.v = (const uint16_t*)p->v;
        a.k_tok = p->k_token; a.k_head = p->k_head;
        a.v_tok = p->v_token; a.v_head = p->v_head;
        a.slots = p->slots;
        a.places = p->places;
        a.hkv = o.num_kv_heads;
        a.kp = (uint16_t*)o.k + p->layer * o.k_layer;
        a.vp = (uint16_t*)o.v + p->layer * o.v_layer;
        a.kp_page = o.k_page; a.kp_head = o.k_head;
        a.vp_page = o.v_page; a.vp_head = o.v_head;
        a.table = p->table;
        a.table_row = p->table_row;
        a.slots_n = p->num_slots;
        a.cols = p->table_cols;
        a.pages = o.num_pages;
        a.page = o.page_size;
        a.shift = __builtin_ctz((unsigned)o.page_size);
        odd |= (p->k_token | p->k_head | p->v_token | p->v_head) % 8;
        vec = vec && al16(p->k) && al16(p->v);
    }
    vec = vec && odd == 0;
    return p->dtype == MQ_BF16 ? run_rope<__nv_bfloat16>(p, a, vec, st) : run_rope<__half>(p, a, vec, st);
}
