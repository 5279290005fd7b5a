// What the C-ABI translation units share: the error string, launch helpers, tensor-map construction, device facts and the
// workspace check.
#pragma once
#include "xs_moe.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <string>
#include <utility>
#include <vector>

namespace xs_api {

inline thread_local std::string g_last_error;

// kernels this library has enqueued since the process started (captured launches count once, at capture)
inline std::atomic<unsigned long long> g_launches{0};
inline void note_launch()
{
    g_launches.fetch_add(1, std::memory_order_relaxed);
}

// Launch with the programmatic-serialisation attribute (see pdl_wait in xs_ptx.cuh): only for kernels whose every thread
// calls xs::pdl_wait() before its first access to global memory that other kernels of the stream write or read.
// XS_MOE_PDL=0 in the environment turns the attribute off (the kernels then start after their predecessor, as usual).
inline bool pdl_enabled()
{
    static const bool on = [] {
        const char *e = getenv("XS_MOE_PDL");
        return !(e && e[0] == '0');
    }();
    return on;
}
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args &&...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, KArgs(std::forward<Args>(args))...);
}

inline int fail(int status, const char *fmt, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_last_error = buf;
    return status;
}

#define XS_CUDA(call)                                                                                       \
    do {                                                                                                    \
        cudaError_t err__ = (call);                                                                         \
        if (err__ != cudaSuccess)                                                                           \
            return fail(XS_MOE_ERR_CUDA, "CUDA error: %s (%s) at %s:%d", cudaGetErrorString(err__), #call, \
                        __FILE__, __LINE__);                                                                \
    } while (0)

inline size_t align_up(size_t v, size_t a)
{
    return (v + a - 1) / a * a;
}

// ---- driver entry point for tensor maps (no link-time dependency on libcuda) ---------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn get_encode_fn()
{
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

// Encoded maps are kept: a layer call describes the same weight matrices (and, with a reused workspace, the same
// activation buffers) every time, and an encode costs about a microsecond of host time -- a tenth of a decode step's launch
// budget when a call needs eight of them.  The key is everything the encoding depends on, so a cached map is exactly the map
// a fresh encode would give.  Small, linear, thread-safe; the oldest entry is replaced when it is full.
struct TmapKey {
    uintptr_t base;
    uint64_t d0, d1, s0;
    uint32_t b0, b1;
    int32_t dt, swizzle, l2;
    bool operator==(const TmapKey &o) const
    {
        return base == o.base && d0 == o.d0 && d1 == o.d1 && s0 == o.s0 && b0 == o.b0 && b1 == o.b1 && dt == o.dt && swizzle == o.swizzle &&
               l2 == o.l2;
    }
};
inline CUresult encode_2d_cached(EncodeTiledFn fn, CUtensorMap *m, CUtensorMapDataType dt, const void *base, const cuuint64_t *dims,
                          const cuuint64_t *strides, const cuuint32_t *box, CUtensorMapSwizzle swz, CUtensorMapL2promotion l2)
{
    constexpr int kEntries = 128;
    struct Entry {
        TmapKey key;
        CUtensorMap map;
    };
    static std::mutex mu;
    static std::vector<Entry> table;
    static size_t next = 0;
    const TmapKey key{reinterpret_cast<uintptr_t>(base), dims[0], dims[1], strides[0], box[0], box[1], static_cast<int32_t>(dt),
                      static_cast<int32_t>(swz), static_cast<int32_t>(l2)};
    {
        std::lock_guard<std::mutex> lock(mu);
        for (const Entry &e : table)
            if (e.key == key) {
                *m = e.map;
                return CUDA_SUCCESS;
            }
    }
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(m, dt, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz, l2,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) {
        std::lock_guard<std::mutex> lock(mu);
        if (table.size() < kEntries) {
            table.push_back(Entry{key, *m});
        } else {
            table[next] = Entry{key, *m};
            next = (next + 1) % kEntries;
        }
    }
    return r;
}

// 2-D row-major matrix (rows, cols) of `elem_bytes`-wide elements; box = (box_cols, box_rows); 128-byte swizzle.
inline int make_tmap_2d(CUtensorMap *m, CUtensorMapDataType dt, int elem_bytes, const void *base, uint64_t rows, uint64_t cols,
                 uint32_t box_rows, uint32_t box_cols)
{
    EncodeTiledFn fn = get_encode_fn();
    if (!fn)
        return fail(XS_MOE_ERR_CUDA, "CUDA error: cuTensorMapEncodeTiled entry point not available");
    if (reinterpret_cast<uintptr_t>(base) % 16 != 0 || (cols * elem_bytes) % 16 != 0)
        return fail(XS_MOE_ERR_INVALID_ARG, "tensor map operand must be 16-byte aligned with a 16-byte multiple row pitch");
    if (box_cols * elem_bytes != 128)
        return fail(XS_MOE_ERR_INVALID_ARG, "internal: swizzled box must be 128 bytes wide");
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {cols * static_cast<uint64_t>(elem_bytes)};
    cuuint32_t box[2] = {box_cols, box_rows};
    CUresult r = encode_2d_cached(fn, m, dt, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (r != CUDA_SUCCESS)
        return fail(XS_MOE_ERR_CUDA, "CUDA error: cuTensorMapEncodeTiled failed with code %d (rows=%llu cols=%llu)", (int)r,
                    (unsigned long long)rows, (unsigned long long)cols);
    return 0;
}

// 2-D row-major byte matrix (rows, row_bytes) read in boxes of (box_bytes, box_rows) WITHOUT swizzle: rows of the box land
// back to back in shared memory.
inline int make_tmap_bytes(CUtensorMap *m, const void *base, uint64_t rows, uint64_t row_bytes, uint32_t box_rows, uint32_t box_bytes)
{
    EncodeTiledFn fn = get_encode_fn();
    if (!fn)
        return fail(XS_MOE_ERR_CUDA, "CUDA error: cuTensorMapEncodeTiled entry point not available");
    if (reinterpret_cast<uintptr_t>(base) % 16 != 0 || row_bytes % 16 != 0 || box_bytes % 16 != 0)
        return fail(XS_MOE_ERR_INVALID_ARG, "tensor map operand must be 16-byte aligned with a 16-byte multiple row pitch");
    cuuint64_t dims[2] = {row_bytes, rows};
    cuuint64_t strides[1] = {row_bytes};
    cuuint32_t box[2] = {box_bytes, box_rows};
    CUresult r = encode_2d_cached(fn, m, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE,
                                  CU_TENSOR_MAP_L2_PROMOTION_NONE);
    if (r != CUDA_SUCCESS)
        return fail(XS_MOE_ERR_CUDA, "CUDA error: cuTensorMapEncodeTiled failed with code %d (rows=%llu row bytes=%llu)", (int)r,
                    (unsigned long long)rows, (unsigned long long)row_bytes);
    return 0;
}

struct DeviceInfo {
    int sms = 0;
    int max_smem = 0;
};

inline int device_info(DeviceInfo *out)
{
    int dev = 0;
    XS_CUDA(cudaGetDevice(&dev));
    // written before `known` says so: a second thread's first call must not see half of it
    static DeviceInfo cache[64];
    static std::atomic<bool> known[64];
    static std::mutex mu;
    if (dev < 64 && known[dev].load(std::memory_order_acquire)) {
        *out = cache[dev];
        return 0;
    }
    int major = 0, sms = 0, smem = 0;
    XS_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
    XS_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    XS_CUDA(cudaDeviceGetAttribute(&smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev));
    if (major != 10)
        return fail(XS_MOE_ERR_DEVICE, "this library holds sm_100a kernels only; device %d has compute capability %d.x", dev, major);
    DeviceInfo d;
    d.sms = sms;
    d.max_smem = smem;
    if (dev < 64) {
        std::lock_guard<std::mutex> lock(mu);
        if (!known[dev].load(std::memory_order_relaxed)) {
            cache[dev] = d;
            known[dev].store(true, std::memory_order_release);
        }
    }
    *out = d;
    return 0;
}

constexpr size_t kStatusBytes = 256; // head of every workspace: the status word the kernels OR into, counters

inline int check_workspace(const void *ws, size_t have, size_t need)
{
    if (!ws)
        return fail(XS_MOE_ERR_WORKSPACE, "workspace is null");
    if (reinterpret_cast<uintptr_t>(ws) % 256 != 0)
        return fail(XS_MOE_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    if (have < need)
        return fail(XS_MOE_ERR_WORKSPACE, "workspace too small: %zu bytes given, %zu needed", have, need);
    return 0;
}

} // namespace xs_api
