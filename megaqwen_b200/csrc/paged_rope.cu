// Rotary positions fused with the write of K and V into the paged cache, and
// the pages' score index.
//
// Memory-bound: each token's q, k and v are read once and written once,
// (Hq + 2 Hkv) D elements each way; the cos/sin row of a token is shared by its
// heads.  One CTA per token: a thread keeps one 16-channel unit's cos/sin in
// registers and walks over heads with it, so the tables cost one read per
// thread and not one per head.
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
    int slots_n, cols, pages, page;
    int* status;
};

// The products and sums are rounded one by one (no FMA), so the result is that
// of the plain formula in fp32 and not of the compiler's contraction.
__device__ __forceinline__ void turn(float& x0, float& x1, float c, float s) {
    const float a = x0, b = x1;
    x0 = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    x1 = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}

// Where token `t` goes.  page -1: nowhere (no cache, or a wrong place).
struct Place {
    int pos, page, row;
    bool ok;   // the position is inside the tables
};
__device__ __forceinline__ Place place_of(const RopeArgs& a, int t, bool report) {
    Place p;
    p.pos = a.positions[t];
    p.page = -1;
    p.row = 0;
    p.ok = p.pos >= 0 && p.pos < a.max_pos;
    if (!p.ok) {
        if (report) note_status(a.status, MQ_ERR_BAD_POSITION);
    } else if (a.kp) {
        const int slot = a.slots[t], c = p.pos / a.page;
        if (slot < 0 || slot >= a.slots_n) {
            if (report) note_status(a.status, MQ_ERR_BAD_SLOT);
        } else if (c >= a.cols) {
            if (report) note_status(a.status, MQ_ERR_BAD_POSITION);
        } else {
            const int g = a.table[slot * a.table_row + c];
            if (g >= 0 && g < a.pages) {
                p.page = g;
                p.row = p.pos - c * a.page;
            } else if (report) {
                note_status(a.status, MQ_ERR_BAD_PAGE);
            }
        }
    }
    return p;
}

// Head h of the token: q heads first, then k, then v.  Sets the pointers;
// false when nothing is to be written.
__device__ __forceinline__ bool head_of(const RopeArgs& a, int t, int h, int D, const Place& p, const uint16_t*& src,
                                        uint16_t*& dst, bool& rotate) {
    if (h < a.hq) {
        src = a.q + t * a.q_tok + h * a.q_head;
        dst = a.q_out + t * a.o_tok + h * a.o_head;
        rotate = true;
        return true;
    }
    if (p.page < 0) return false;
    const int g = h - a.hq;
    if (g < a.hkv) {
        src = a.k + t * a.k_tok + g * a.k_head;
        dst = a.kp + p.page * a.kp_page + g * a.kp_head + p.row * D;
        rotate = true;
    } else {
        src = a.v + t * a.v_tok + (g - a.hkv) * a.v_head;
        dst = a.vp + p.page * a.vp_page + (g - a.hkv) * a.vp_head + p.row * D;
        rotate = false;
    }
    return true;
}

// Vector path: rotary_dim a multiple of 16, every address a multiple of 16
// bytes.  A unit is 16 channels of a head: for the half layout the 8 pairs
// (8u + i, 8u + i + R / 2), otherwise 16 channels in a row.
template <typename T, int D, bool INTER>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const RopeArgs a) {
    constexpr int UNITS = D / 16, LANES = ROPE_THREADS / UNITS;
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x, u = threadIdx.x % UNITS;
    const Place p = place_of(a, t, threadIdx.x == 0);
    const bool rot_unit = u < a.rot / 16;
    const int heads = a.hq + (a.kp ? 2 * a.hkv : 0);
    // first channels of the unit's two 8-channel pieces
    const int c0 = !INTER && rot_unit ? 8 * u : 16 * u;
    const int c1 = !INTER && rot_unit ? 8 * u + a.rot / 2 : 16 * u + 8;
    const int r0 = c0, r1 = rot_unit && !INTER ? c1 : c0 + 8;
    // pieces of a v head (never rotated) are taken in the same places: a permutation of the units
    float cs[8], sn[8];
    if (rot_unit && p.ok) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(a.cos_t + p.pos * a.cos_row + 8 * u + i);
            const float4 y = *reinterpret_cast<const float4*>(a.sin_t + p.pos * a.sin_row + 8 * u + i);
            cs[i] = x.x; cs[i + 1] = x.y; cs[i + 2] = x.z; cs[i + 3] = x.w;
            sn[i] = y.x; sn[i + 1] = y.y; sn[i + 2] = y.z; sn[i + 3] = y.w;
        }
        if (a.inverse) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sn[i] = -sn[i];
        }
    }
#pragma unroll 2
    for (int h = threadIdx.x / UNITS; h < heads; h += LANES) {
        const uint16_t* src;
        uint16_t* dst;
        bool rotate;
        if (!head_of(a, t, h, D, p, src, dst, rotate)) continue;
        uint4 x = *reinterpret_cast<const uint4*>(src + r0), y = *reinterpret_cast<const uint4*>(src + r1);
        if (!p.ok) x = y = make_uint4(0, 0, 0, 0);   // a position outside the tables has no rotation
        if (rotate && rot_unit && p.ok) {
            uint32_t* xv = reinterpret_cast<uint32_t*>(&x);
            uint32_t* yv = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 e = Elem<T>::up2(xv[i]), f = Elem<T>::up2(yv[i]);
                if (INTER) {   // pairs are neighbours: x holds pairs 8u .. 8u + 3, y the next four
                    turn(e.x, e.y, cs[i], sn[i]);
                    turn(f.x, f.y, cs[4 + i], sn[4 + i]);
                } else {
                    turn(e.x, f.x, cs[2 * i], sn[2 * i]);
                    turn(e.y, f.y, cs[2 * i + 1], sn[2 * i + 1]);
                }
                xv[i] = Elem<T>::pack(e.x, e.y);
                yv[i] = Elem<T>::pack(f.x, f.y);
            }
        }
        *reinterpret_cast<uint4*>(dst + r0) = x;
        *reinterpret_cast<uint4*>(dst + r1) = y;
    }
}

// Any even rotary_dim and any alignment: a thread per pair of channels.
template <typename T>
__global__ void __launch_bounds__(ROPE_THREADS) rope_any_kernel(const RopeArgs a, int D, int inter) {
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x, half = a.rot / 2;
    const Place p = place_of(a, t, threadIdx.x == 0);
    const int heads = a.hq + (a.kp ? 2 * a.hkv : 0);
    for (int e = threadIdx.x; e < heads * (D / 2); e += ROPE_THREADS) {
        const int h = e / (D / 2), i = e - h * (D / 2);
        const uint16_t* src;
        uint16_t* dst;
        bool rotate;
        if (!head_of(a, t, h, D, p, src, dst, rotate)) continue;
        const bool in = i < half;
        const int c0 = in && !inter ? i : 2 * i, c1 = in && !inter ? i + half : 2 * i + 1;
        uint16_t x = src[c0], y = src[c1];
        if (!p.ok) x = y = 0;
        if (rotate && in && p.ok) {
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
// CTA (chunk of 128 tokens, kv head): for each token of the chunk that is the
// last row of its page, the bounds of the page's keys over its rows (read from
// L2, where the kernel before left them).  Bounds are exact (no arithmetic on
// the keys), so the record does not depend on the order of the rows.
constexpr int INDEX_THREADS = 256, INDEX_TOKENS = 128;

template <typename T, int D>
__global__ void __launch_bounds__(INDEX_THREADS) index_kernel(const RopeArgs a, int n, signed char* __restrict__ index,
                                                              long long i_page, long long i_head) {
    constexpr int PIECES = D / 8, ROWS = INDEX_THREADS / PIECES;   // 8 channels a thread, ROWS rows at once
    __shared__ int list[INDEX_TOKENS];
    __shared__ int count;
    __shared__ float red[2][ROWS][D];
    __shared__ float amax[D / 32];
    pdl_wait();
    pdl_trigger();
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const int t = blockIdx.x * INDEX_TOKENS + threadIdx.x, h = blockIdx.y;
    if (threadIdx.x < INDEX_TOKENS && t < n && a.positions[t] % a.page == a.page - 1) {
        const Place p = place_of(a, t, false);
        if (p.page >= 0) list[atomicAdd(&count, 1)] = p.page;
    }
    __syncthreads();
    const int piece = threadIdx.x % PIECES, r0 = threadIdx.x / PIECES;
    for (int e = 0; e < count; ++e) {
        const uint16_t* k = a.kp + list[e] * a.kp_page + h * a.kp_head;
        float hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            hi[i] = -INFINITY;
            lo[i] = INFINITY;
        }
        for (int r = r0; r < a.page; r += ROWS) {
            const uint4 x = *reinterpret_cast<const uint4*>(k + r * D + piece * 8);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = Elem<T>::up2(w[i]);
                hi[2 * i] = fmaxf(hi[2 * i], f.x);
                lo[2 * i] = fminf(lo[2 * i], f.x);
                hi[2 * i + 1] = fmaxf(hi[2 * i + 1], f.y);
                lo[2 * i + 1] = fminf(lo[2 * i + 1], f.y);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            red[0][r0][piece * 8 + i] = hi[i];
            red[1][r0][piece * 8 + i] = lo[i];
        }
        __syncthreads();
        float H = -INFINITY, L = INFINITY;
        const int d = threadIdx.x;
        if (d < D) {
            for (int r = 0; r < ROWS; ++r) {
                H = fmaxf(H, red[0][r][d]);
                L = fminf(L, red[1][r][d]);
            }
            // infinite keys count as the type's largest, and a channel of nothing but NaN as zero
            if (!(H >= L)) H = L = 0.f;
            H = fminf(fmaxf(H, -Elem<T>::MAX), Elem<T>::MAX);
            L = fminf(fmaxf(L, -Elem<T>::MAX), Elem<T>::MAX);
            float m = fmaxf(fabsf(H), fabsf(L));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if ((d & 31) == 0) amax[d >> 5] = m;
        }
        __syncthreads();
        if (d < D) {
            float m = amax[0];
#pragma unroll
            for (int i = 1; i < D / 32; ++i) m = fmaxf(m, amax[i]);
            const int ex = m > 0.f ? min(max(ilogbf(m) - 6, -60), 40) : 0;
            const float unit = __int_as_float((127 - ex) << 23);   // 2^-ex
            signed char* rec = index + list[e] * i_page + h * i_head;
            rec[d] = (signed char)fminf(fmaxf(rintf(H * unit), -127.f), 127.f);
            rec[D + d] = (signed char)fminf(fmaxf(rintf(L * unit), -127.f), 127.f);
            if (d < 16) rec[2 * D + d] = d == 0 ? (signed char)ex : 0;
        }
        __syncthreads();
    }
}

template <typename T>
int run_rope(const mq_rope_params* p, const RopeArgs& a, bool vec, cudaStream_t st) {
    const int D = p->head_dim;
    cudaError_t e;
    if (!vec)
        e = launch(rope_any_kernel<T>, dim3(p->n), dim3(ROPE_THREADS), 0, st, a, D, p->interleaved);
    else if (D == 128)
        e = p->interleaved ? launch(rope_kernel<T, 128, true>, dim3(p->n), dim3(ROPE_THREADS), 0, st, a)
                           : launch(rope_kernel<T, 128, false>, dim3(p->n), dim3(ROPE_THREADS), 0, st, a);
    else
        e = p->interleaved ? launch(rope_kernel<T, 64, true>, dim3(p->n), dim3(ROPE_THREADS), 0, st, a)
                           : launch(rope_kernel<T, 64, false>, dim3(p->n), dim3(ROPE_THREADS), 0, st, a);
    if (e != cudaSuccess) return note_cuda(e, "rope");
    if (!p->pool || !p->pool->index) return MQ_OK;
    signed char* ix = p->pool->index + p->layer * p->pool->i_layer;
    const dim3 grid(ceil_div(p->n, INDEX_TOKENS), p->pool->num_kv_heads);
    e = D == 128 ? launch(index_kernel<T, 128>, grid, dim3(INDEX_THREADS), 0, st, a, p->n, ix, p->pool->i_page, p->pool->i_head)
                 : launch(index_kernel<T, 64>, grid, dim3(INDEX_THREADS), 0, st, a, p->n, ix, p->pool->i_page, p->pool->i_head);
    return e == cudaSuccess ? MQ_OK : note_cuda(e, "page index");
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
        odd |= (p->k_token | p->k_head | p->v_token | p->v_head) % 8;
        vec = vec && al16(p->k) && al16(p->v);
    }
    vec = vec && odd == 0;
    return p->dtype == MQ_BF16 ? run_rope<__nv_bfloat16>(p, a, vec, st) : run_rope<__half>(p, a, vec, st);
}
