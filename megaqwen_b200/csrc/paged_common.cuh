// What the paged-cache kernels share: the two 16-bit element types, the pool's
// address arithmetic, the status word and launch helpers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "megaqwen_b200.h"
#include "mq_ptx.cuh"

namespace mq {

int note_cuda(cudaError_t e, const char* what);

namespace paged {

// Element type traits: packing of fp32 pairs and the mma.sync flavour.
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float up(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&t);
    }
    static __device__ __forceinline__ float2 up2(uint32_t v) { return make_float2(bf16lo(v), bf16hi(v)); }
    static __device__ __forceinline__ uint16_t down(float x) { return __bfloat16_as_ushort(__float2bfloat16(x)); }
    static constexpr uint32_t EXP_MASK = 0x7f80u;   // all ones: infinity or NaN
    static constexpr float MAX = 3.3895313892515355e38f;
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float up(uint16_t x) { return __half2float(__ushort_as_half(x)); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        __half2 t = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&t);
    }
    static __device__ __forceinline__ float2 up2(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
    static __device__ __forceinline__ uint16_t down(float x) { return __half_as_ushort(__float2half_rn(x)); }
    static constexpr uint32_t EXP_MASK = 0x7c00u;
    static constexpr float MAX = 65504.f;
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// The first error stays in the status word; later calls do not overwrite it.
__device__ __forceinline__ void note_status(int* status, int code) {
    if (status) atomicCAS(status, 0, code);
}

__host__ __device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
// pages that hold `len` positions; exact up to the largest int
__host__ __device__ __forceinline__ int pages_of(int len, int page) { return len <= 0 ? 0 : (len - 1) / page + 1; }

inline int sm_count() {
    static int sms[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 148;
    if (!sms[dev]) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
    return sms[dev] > 0 ? sms[dev] : 148;
}

// Raises a kernel's shared-memory limit to the largest that the device allows, on
// its first use there (the driver call is worth avoiding in a call of a few
// microseconds).  `set` is the kernel's own record, one entry per device: the limit
// that is in place.  Every thread that gets to set it sets the same, so it does not
// matter who is first.
struct SmemLimit {
    std::atomic<int> bytes[64];
};
template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes, SmemLimit& set) {
    int dev = 0, most = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64) most = set.bytes[dev].load(std::memory_order_relaxed);
    if (!most) {
        cudaFuncAttributes at;
        e = cudaFuncGetAttributes(&at, kernel);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
        if (e != cudaSuccess) return e;
        most -= (int)at.sharedSizeBytes;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
        if (dev < 64) set.bytes[dev].store(most, std::memory_order_relaxed);
    }
    return bytes <= (size_t)most ? cudaSuccess : cudaErrorInvalidValue;
}

// Thread-block clusters of the one-dimensional grids here.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();   // the aligned form takes whole warps
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_peer(uint32_t addr, uint32_t rank, uint32_t v) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

__device__ __forceinline__ void red_peer_max(uint32_t addr, uint32_t rank, int v) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    asm volatile("red.relaxed.cluster.shared::cluster.max.s32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

// Every kernel here is launched as a programmatic dependent of the kernel
// before it in the stream and begins with pdl_wait, so stream order holds and
// only the launch itself overlaps the previous kernel's tail.
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, ((KArgs)args)...);
}

// The same in clusters of `ranks` CTAs.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), unsigned grid, unsigned ranks, dim3 block, size_t smem, cudaStream_t st,
                           Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, ((KArgs)args)...);
}

// The index records of the pages whose last row is one of the n positions, in every layer (paged_rope.cu).
int reindex(const mq_paged_pool* pool, const int* table, long long table_row, int num_slots, int cols, const int* positions,
            const int* slots, int n, cudaStream_t st);

inline bool pool_ok(const mq_paged_pool* p) {
    return p && p->k && p->v && (p->dtype == MQ_BF16 || p->dtype == MQ_FP16) && p->num_pages >= 1 && p->num_layers >= 1 &&
           p->num_kv_heads >= 1 && p->num_kv_heads <= 1024 && (p->head_dim == 64 || p->head_dim == 128) &&
           (p->page_size == 16 || p->page_size == 32 || p->page_size == 64 || p->page_size == 128) &&
           (reinterpret_cast<uintptr_t>(p->k) & 15) == 0 && (reinterpret_cast<uintptr_t>(p->v) & 15) == 0 &&
           p->k_page % 8 == 0 && p->k_layer % 8 == 0 && p->k_head % 8 == 0 && p->v_page % 8 == 0 &&
           p->v_layer % 8 == 0 && p->v_head % 8 == 0 &&
           (!p->index || ((reinterpret_cast<uintptr_t>(p->index) & 15) == 0 && p->i_page % 16 == 0 &&
                          p->i_layer % 16 == 0 && p->i_head % 16 == 0));
}

}  // namespace paged
}  // namespace mq
