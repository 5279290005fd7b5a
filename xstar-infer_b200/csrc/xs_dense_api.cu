// C ABI of include/xs_moe_dense.h: argument checks, workspace plans and launches.  No exception leaves this file.
#include "xs_moe_dense.h"

#include <atomic>

#include "xs_api_common.cuh"
#include "xs_norm_residual.cuh"
#include "xs_w4_prepare.cuh"
#include "xs_w4_small.cuh"
#include "xs_w4_tc.cuh"

using namespace xs_api;

namespace {

// A pointer the kernels may follow: device (or managed) memory of the current device.
int check_on_device(const void *p, int device, const char *name)
{
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        return fail(XS_MOE_ERR_INVALID_ARG, "device mismatch: %s is not device memory", name);
    }
    if (at.type == cudaMemoryTypeManaged)
        return 0;
    if (at.type != cudaMemoryTypeDevice)
        return fail(XS_MOE_ERR_INVALID_ARG, "device mismatch: %s is not device memory", name);
    if (at.device != device)
        return fail(XS_MOE_ERR_INVALID_ARG, "device mismatch: %s is on device %d, the current device is %d", name, at.device, device);
    return 0;
}

int current_device(int *dev)
{
    XS_CUDA(cudaGetDevice(dev));
    return 0;
}

bool overlap(const void *a, size_t an, const void *b, size_t bn)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && an && bn && x < y + bn && y < x + an;
}

bool misaligned(const void *p, uintptr_t n)
{
    return reinterpret_cast<uintptr_t>(p) % n != 0;
}

constexpr int32_t kMaxDim = 1 << 30; // the kernels round sizes up to whole tiles in 32 bits

// shapes only: what the workspace queries need
int check_w4_shape(const XsMoeW4 *w, int32_t tokens)
{
    if (!w)
        return fail(XS_MOE_ERR_INVALID_ARG, "weight is null");
    if (w->reserved != 0)
        return fail(XS_MOE_ERR_INVALID_ARG, "reserved fields must be zero");
    if (tokens < 0 || w->rows <= 0 || w->cols <= 0)
        return fail(XS_MOE_ERR_INVALID_ARG, "shape mismatch: non-positive dimension");
    if (tokens > kMaxDim || w->rows > kMaxDim || w->cols > kMaxDim)
        return fail(XS_MOE_ERR_UNSUPPORTED, "rows, columns and tokens must be at most 2^30");
    if (w->group != 32 && w->group != 64 && w->group != 128)
        return fail(XS_MOE_ERR_UNSUPPORTED, "group must be 32, 64 or 128");
    if (w->cols % w->group != 0)
        return fail(XS_MOE_ERR_INVALID_ARG, "shape mismatch: columns must be a multiple of the group");
    return 0;
}

int check_gated_shape(const XsMoeW4 *w, int32_t activation, int32_t tokens)
{
    if (int rc = check_w4_shape(w, tokens))
        return rc;
    if (w->rows % 2 != 0)
        return fail(XS_MOE_ERR_INVALID_ARG, "gate_up out must be even");
    if (activation != XS_MOE_SILU && activation != XS_MOE_GELU_TANH)
        return fail(XS_MOE_ERR_UNSUPPORTED, "unknown activation");
    return 0;
}

int check_mlp_shape(const XsMoeW4 *gu, const XsMoeW4 *dn, int32_t activation, int32_t tokens)
{
    if (int rc = check_gated_shape(gu, activation, tokens))
        return rc;
    if (int rc = check_w4_shape(dn, tokens))
        return rc;
    if (dn->cols != gu->rows / 2 || dn->rows != gu->cols)
        return fail(XS_MOE_ERR_INVALID_ARG, "shape mismatch: down must be (hidden, intermediate)");
    return 0;
}

// out, ws: what the call writes, which must not be what it reads
int check_w4_data(const XsMoeW4 *w, const void *out, size_t out_elems, const void *ws, size_t ws_bytes, int dev)
{
    if (!w->codes_dev || !w->scales_dev)
        return fail(XS_MOE_ERR_INVALID_ARG, "null tensor pointer");
    if (misaligned(w->codes_dev, 16) || misaligned(w->scales_dev, 2))
        return fail(XS_MOE_ERR_INVALID_ARG, "tensors must be 16-byte aligned (scales 2-byte)");
    const size_t rows = w->rows, groups = w->cols / w->group;
    const void *ptr[] = {w->codes_dev, w->scales_dev, w->zeros_dev};
    const size_t bytes[] = {rows * w->cols / 2, rows * groups * 2, rows * groups};
    for (int i = 0; i < 3; i++)
        if (overlap(ptr[i], bytes[i], out, out_elems * 2) || overlap(ptr[i], bytes[i], ws, ws_bytes))
            return fail(XS_MOE_ERR_INVALID_ARG, "a weight overlaps out or the workspace");
    if (int rc = check_on_device(w->codes_dev, dev, "codes"))
        return rc;
    if (int rc = check_on_device(w->scales_dev, dev, "scales"))
        return rc;
    return w->zeros_dev ? check_on_device(w->zeros_dev, dev, "zeros") : 0;
}

// in_place: the caller may write the result over x itself (same address)
int check_io(const void *x, size_t x_elems, void *out, size_t out_elems, const void *ws, size_t ws_bytes, int dev, bool in_place = false)
{
    if (!x || !out)
        return fail(XS_MOE_ERR_INVALID_ARG, "null tensor pointer");
    if (misaligned(x, 16) || misaligned(out, 2))
        return fail(XS_MOE_ERR_INVALID_ARG, "x must be 16-byte aligned, out 2-byte");
    if ((!(in_place && x == out) && overlap(x, x_elems * 2, out, out_elems * 2)) || overlap(x, x_elems * 2, ws, ws_bytes) || overlap(out, out_elems * 2, ws, ws_bytes))
        return fail(XS_MOE_ERR_INVALID_ARG, "x, out and the workspace must not overlap");
    if (int rc = check_on_device(x, dev, "x"))
        return rc;
    if (int rc = check_on_device(out, dev, "out"))
        return rc;
    return check_on_device(ws, dev, "workspace");
}

size_t bf16_bytes(size_t rows, size_t cols)
{
    return align_up(rows * cols * 2, 256);
}

xs::W4Matrix matrix_of(const XsMoeW4 *w)
{
    return {static_cast<const uint8_t *>(w->codes_dev), static_cast<const __nv_bfloat16 *>(w->scales_dev), w->zeros_dev};
}

// The codes as `parts` byte matrices one after the other (gate and up, or one), read in boxes of 128 bytes x box_rows of
// each, 128-byte swizzle; bytes and rows past the end read as zero.
int make_tmap_codes(CUtensorMap *m, const XsMoeW4 *w, int parts, uint32_t box_rows)
{
    EncodeTiledFn fn = get_encode_fn();
    if (!fn)
        return fail(XS_MOE_ERR_CUDA, "CUDA error: cuTensorMapEncodeTiled entry point not available");
    const cuuint64_t bytes = static_cast<cuuint64_t>(w->cols) / 2, rows = static_cast<cuuint64_t>(w->rows) / parts;
    const cuuint64_t dims[3] = {bytes, rows, static_cast<cuuint64_t>(parts)}, strides[2] = {bytes, bytes * rows};
    const cuuint32_t box[3] = {128, box_rows, static_cast<cuuint32_t>(parts)}, one[3] = {1, 1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(w->codes_dev), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(XS_MOE_ERR_CUDA, "CUDA error: cuTensorMapEncodeTiled failed with code %d (rows=%d cols=%d)", (int)r, w->rows, w->cols);
    return 0;
}

// The shared memory that a kernel may ask for, set once for each device, to the most that any of its launches takes: two threads
// that set it to what their own call needs would undo one another's.
struct SmemLimit {
    std::atomic<uint64_t> done{0};
    template <typename Kernel>
    int set(Kernel *kern, int bytes)
    {
        int dev = 0;
        XS_CUDA(cudaGetDevice(&dev));
        const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
        if (!(done.load(std::memory_order_acquire) & bit)) {
            XS_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
            done.fetch_or(bit, std::memory_order_release);
        }
        return 0;
    }
};

// A programmatic dependent launch in clusters of `cluster` blocks.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl_cluster(void (*kern)(KArgs...), int grid, int block, int cluster, size_t smem, cudaStream_t st, Args &&...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, KArgs(std::forward<Args>(args))...);
}

// How many clusters of 1, 2, 4 and 8 blocks, each block with an SM to itself, run at one time.  A cluster lies within a GPC, so this is
// less than the SMs would give: the grid of a plan with one cluster more than that takes twice as long (294 x 2816 x 1516
// with 36 clusters of four: 22.8 us; planned with what fits: 14.3).
struct ClusterSlots {
    int of[4];
    int operator()(int cluster) const
    {
        return of[cluster == 1 ? 0 : cluster == 2 ? 1 : cluster == 4 ? 2 : 3];
    }
};

int cluster_slots(const DeviceInfo &di, ClusterSlots *out)
{
    static std::atomic<int> known[64][4];
    int dev = 0;
    XS_CUDA(cudaGetDevice(&dev));
    out->of[0] = di.sms;
    auto kern = xs::w4_small_kernel<false, 4, false, false, 1>;
    for (int i = 1; i < 4; i++) {
        int n = dev < 64 ? known[dev][i].load(std::memory_order_relaxed) : 0;
        if (n == 0) {
            XS_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, di.max_smem));
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = di.sms / (1 << i) * (1 << i);
            cfg.blockDim = 32 * xs::kSwWarps;
            cfg.dynamicSmemBytes = di.max_smem;
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 1 << i;
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            XS_CUDA(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
            n = n < 1 ? 1 : n;
            if (dev < 64)
                known[dev][i].store(n, std::memory_order_relaxed);
        }
        out->of[i] = n;
    }
    return 0;
}

struct SmallPlan {
    int ways = 1, cluster = 1, chunks_per_block = 0, stages = 2, grid = 0, smem = 0;
};

// How the warps share the work: `ways` warps of a block on the same rows, `cluster` blocks on the same tile.  Taken is what gives
// the busiest block the least work, counted in chunks of a warp; a tile's sum, barrier and store take about as long as
// kTileCost of them, a cluster's kClusterCost more.
SmallPlan plan_small(int T, int K, int n_out, int band_rows, const ClusterSlots &slots, int max_smem)
{
    constexpr float kTileCost = 0.4f, kClusterCost = 0.6f;
    const int chunks = (K + xs::kSwChunk - 1) / xs::kSwChunk;
    SmallPlan best;
    float best_cost = 0.0f;
    for (int c = 1; c <= 8; c *= 2) {
        SmallPlan p;
        p.cluster = c;
        p.chunks_per_block = (chunks + c - 1) / c;
        if (c > 1 && p.chunks_per_block * (c - 1) >= chunks)
            break; // a block would have none
        if (xs::sw_smem_bytes(T, p.chunks_per_block, 2) > max_smem)
            continue;
        for (p.stages = xs::kSwMaxStages; xs::sw_smem_bytes(T, p.chunks_per_block, p.stages) > max_smem; p.stages--) {
        }
        p.smem = static_cast<int>(xs::sw_smem_bytes(T, p.chunks_per_block, p.stages));
        for (p.ways = xs::kSwWarps; p.ways >= 1; p.ways /= 2) {
            const int tiles = (n_out + xs::kSwWarps / p.ways * band_rows - 1) / (xs::kSwWarps / p.ways * band_rows);
            const int clusters = tiles < slots(c) ? tiles : slots(c), rounds = (tiles + clusters - 1) / clusters;
            const int per_warp = (p.chunks_per_block + p.ways - 1) / p.ways;
            const float cost = rounds * (per_warp + kTileCost + (c > 1 ? kClusterCost : 0.0f));
            if (best.grid == 0 || cost < best_cost) {
                best = p;
                best.grid = clusters * c;
                best_cost = cost;
            }
        }
    }
    return best;
}

template <bool GATED, int SUB, bool ZEROS, bool HALF, int NT>
int launch_small_t(const XsMoeW4 *w, const void *x, int T, void *out, int act, bool out_f32, bool early, int32_t *status, cudaStream_t st)
{
    DeviceInfo di;
    if (int rc = device_info(&di))
        return rc;
    const int n_out = GATED ? w->rows / 2 : w->rows;
    ClusterSlots slots;
    if (int rc = cluster_slots(di, &slots))
        return rc;
    const SmallPlan p = plan_small(T, w->cols, n_out, GATED ? 16 : 32, slots, di.max_smem);
    if (p.grid == 0)
        return fail(XS_MOE_ERR_UNSUPPORTED, "internal: no plan for %d tokens of %d columns", T, w->cols);
    CUtensorMap map;
    if (int rc = make_tmap_codes(&map, w, GATED ? 2 : 1, GATED ? 16 : 32))
        return rc;
    auto kern = xs::w4_small_kernel<GATED, SUB, ZEROS, HALF, NT>;
    static SmemLimit limit;
    if (int rc = limit.set(kern, di.max_smem))
        return rc;
    XS_CUDA(launch_pdl_cluster(kern, p.grid, 32 * xs::kSwWarps, p.cluster, p.smem, st, map, matrix_of(w), x, out, n_out, T, w->cols, act, out_f32 ? 1 : 0,
                               early ? 1 : 0, p.ways, p.cluster, p.chunks_per_block, p.stages, status));
    note_launch();
    return 0;
}

template <bool GATED, bool HALF, int NT>
int launch_small_n(const XsMoeW4 *w, const void *x, int T, void *out, int act, bool out_f32, bool early, int32_t *status, cudaStream_t st)
{
    const bool z = w->zeros_dev != nullptr;
    if (w->group == 32)
        return z ? launch_small_t<GATED, 1, true, HALF, NT>(w, x, T, out, act, out_f32, early, status, st)
                 : launch_small_t<GATED, 1, false, HALF, NT>(w, x, T, out, act, out_f32, early, status, st);
    if (w->group == 64)
        return z ? launch_small_t<GATED, 2, true, HALF, NT>(w, x, T, out, act, out_f32, early, status, st)
                 : launch_small_t<GATED, 2, false, HALF, NT>(w, x, T, out, act, out_f32, early, status, st);
    return z ? launch_small_t<GATED, 4, true, HALF, NT>(w, x, T, out, act, out_f32, early, status, st)
             : launch_small_t<GATED, 4, false, HALF, NT>(w, x, T, out, act, out_f32, early, status, st);
}

template <bool GATED, bool HALF>
int launch_small(const XsMoeW4 *w, const void *x, int T, void *out, int act, bool out_f32, bool early, int32_t *status, cudaStream_t st)
{
    return T <= 8 ? launch_small_n<GATED, HALF, 1>(w, x, T, out, act, out_f32, early, status, st)
                  : launch_small_n<GATED, HALF, 2>(w, x, T, out, act, out_f32, early, status, st);
}

// `early` above: nothing that may still be running when the kernel starts writes the weights (it is not the first kernel of its
// call).  One product alone:
int run_small(const XsMoeW4 *w, bool gated, int act, const void *x, int T, void *out, int32_t *status, cudaStream_t st)
{
    return gated ? launch_small<true, false>(w, x, T, out, act, false, false, status, st)
                 : launch_small<false, false>(w, x, T, out, 0, false, false, status, st);
}

// A batch of f16 rows read in boxes of 64 columns x box_rows, 128-byte swizzle; past the end of rows and columns there are zeros.
int make_tmap_rows(CUtensorMap *m, const void *x, int T, int K, uint32_t box_rows)
{
    EncodeTiledFn fn = get_encode_fn();
    if (!fn)
        return fail(XS_MOE_ERR_CUDA, "CUDA error: cuTensorMapEncodeTiled entry point not available");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(T)}, strides[1] = {static_cast<cuuint64_t>(K) * 2};
    const cuuint32_t box[2] = {64, box_rows}, one[2] = {1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(x), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(XS_MOE_ERR_CUDA, "CUDA error: cuTensorMapEncodeTiled failed with code %d (rows=%d cols=%d)", (int)r, T, K);
    return 0;
}

struct TcPlan {
    int cg = 1, n_tile = 32, grid = 0;
    float cost = 0.0f;
    xs::TcShape shape{};
};

// Tile and split by the estimated time of the busiest block, from measurements (microseconds): a 128-column block of a tile takes
// 0.42 with 32 tokens, 0.46 with 64, 0.6 with 128; on a pair of SMs 0.48 with 128 and 0.8 with 256; a tile's start, sums and
// store 2 and 0.006 a token; meeting the other slices of K 1.6 more.
constexpr struct {
    int cg, n_tile;
    float block;
} kTcTiles[] = {{1, 32, 0.42f}, {1, 64, 0.46f}, {1, 128, 0.6f}, {2, 128, 0.48f}, {2, 256, 0.8f}};

// `features` features from f0 on, with one launch; `tile`: one of kTcTiles, or -1 for the best
TcPlan plan_tc_part(const XsMoeW4 *w, bool gated, int T, const ClusterSlots &all, int f0, int features, int tile)
{
    const int n_out = gated ? w->rows / 2 : w->rows, K = w->cols, all_raw = (K + 255) / 256;
    TcPlan best;
    for (int i = 0; i < 5; i++) {
        if (tile >= 0 && i != tile)
            continue;
        const int cg = kTcTiles[i].cg, n_tile = kTcTiles[i].n_tile, width = (gated ? xs::kTcRows / 2 : xs::kTcRows) * cg;
        for (int split = 1; split <= (cg == 1 ? 8 : 1); split *= 2) {
            const int raw_per = (all_raw + split - 1) / split;
            if (raw_per * (split - 1) >= all_raw)
                break;
            TcPlan p;
            p.cg = cg;
            p.n_tile = n_tile;
            p.shape = {n_out, T, K, w->group == 32 ? 5 : w->group == 64 ? 6 : 7, (features + width - 1) / width, (T + n_tile - 1) / n_tile, split, f0};
            const long items = static_cast<long>(p.shape.w_tiles) * p.shape.t_tiles;
            const int slots = all(cg * split);
            if (split > 1 && items > slots)
                break; // a split block has one tile
            const long rounds = (items + slots - 1) / slots;
            p.grid = static_cast<int>(items < slots ? items : slots) * cg * split;
            p.cost = rounds * (raw_per * 2 * kTcTiles[i].block + 2.0f + 0.006f * n_tile) + (split > 1 ? 1.6f : 0.0f);
            if (best.grid == 0 || p.cost < best.cost)
                best = p;
        }
    }
    return best;
}

// One launch, or two: whole rounds of tiles on every SM, and what would have been a last round of few tiles in another shape.
// Returns the number of launches.
int plan_tc(const XsMoeW4 *w, bool gated, int T, const ClusterSlots &all, TcPlan (&plan)[2])
{
    // A second launch starts cold; the estimate has to say that it pays (45 x 4096 x 20480: 38.8 us with it, 42.3 without).
    constexpr float kLaunchCost = 6.0f, kGain = 0.9f;
    const int n_out = gated ? w->rows / 2 : w->rows;
    plan[0] = plan_tc_part(w, gated, T, all, 0, n_out, -1);
    float cost = plan[0].cost;
    int parts = 1;
    for (int i = 0; i < 5; i++) {
        const int cg = kTcTiles[i].cg, n_tile = kTcTiles[i].n_tile, width = (gated ? xs::kTcRows / 2 : xs::kTcRows) * cg, slots = all(cg);
        const long t_tiles = (T + n_tile - 1) / n_tile, items = (n_out + width - 1) / width * t_tiles, rounds = items / slots;
        const int first = static_cast<int>(rounds * slots / t_tiles) * width; // features of the whole rounds
        if (rounds == 0 || first <= 0 || first >= n_out)
            continue;
        const TcPlan a = plan_tc_part(w, gated, T, all, 0, first, i), b = plan_tc_part(w, gated, T, all, first, n_out - first, -1);
        if (a.cost + b.cost + kLaunchCost < cost * (parts == 1 ? kGain : 1.0f)) {
            cost = a.cost + b.cost + kLaunchCost;
            plan[0] = a;
            plan[1] = b;
            parts = 2;
        }
    }
    return parts;
}

template <int CG, int N_TILE, bool GATED, typename Out>
int launch_tc_t(const XsMoeW4 *w, const TcPlan &p, const void *x16, Out *out, const xs::TcOperands &ops, int act, int32_t *status, cudaStream_t st)
{
    auto kern = xs::w4_tc_kernel<CG, N_TILE, GATED, Out>;
    constexpr int smem = xs::tc_smem_bytes(CG, N_TILE);
    static SmemLimit limit;
    if (int rc = limit.set(kern, smem))
        return rc;
    CUtensorMap mw, mx;
    if (int rc = make_tmap_codes(&mw, w, GATED ? 2 : 1, GATED ? xs::kTcRows / 2 : xs::kTcRows))
        return rc;
    if (int rc = make_tmap_rows(&mx, x16, p.shape.T, p.shape.K, N_TILE / CG))
        return rc;
    XS_CUDA(launch_pdl_cluster(kern, p.grid, xs::kTcThreads, CG * p.shape.split, smem, st, mw, mx, ops, out, p.shape, act, status));
    note_launch();
    return 0;
}

template <bool GATED, typename Out>
int launch_tc(const XsMoeW4 *w, const void *x16, int T, Out *out, const xs::TcOperands &ops, int act, int32_t *status, cudaStream_t st)
{
    DeviceInfo di;
    if (int rc = device_info(&di))
        return rc;
    TcPlan plan[2];
    ClusterSlots slots;
    if (int rc = cluster_slots(di, &slots))
        return rc;
    const int parts = plan_tc(w, GATED, T, slots, plan);
    for (int i = 0; i < parts; i++) {
        const TcPlan &p = plan[i];
        int rc = 0;
        if (p.cg == 2 && p.n_tile == 128)
            rc = launch_tc_t<2, 128, GATED, Out>(w, p, x16, out, ops, act, status, st);
        else if (p.cg == 2)
            rc = launch_tc_t<2, 256, GATED, Out>(w, p, x16, out, ops, act, status, st);
        else if (p.n_tile == 128)
            rc = launch_tc_t<1, 128, GATED, Out>(w, p, x16, out, ops, act, status, st);
        else if (p.n_tile == 64)
            rc = launch_tc_t<1, 64, GATED, Out>(w, p, x16, out, ops, act, status, st);
        else
            rc = launch_tc_t<1, 32, GATED, Out>(w, p, x16, out, ops, act, status, st);
        if (rc)
            return rc;
    }
    return 0;
}

// Which kernel: up to sixteen tokens the one that streams weights past the tokens, if a cluster's shared memory holds them.  4096 x
// 4096 with 1, 8, 9, 16 tokens: 5.5, 6.5, 7.7, 8.8 us against 11.3, 11.4, 11.5, 11.8 on the tensor core; 8 x 4096 x 32003 with
// zero points 24 us against 40, 16 tokens 34 against 40.  Clusters of eight do not fill the SMs: more than eight tokens go to the tensor
// core before they take one (16 x 11264 x 4096 with zero points: 22 us against 34; 13 x 16384 x 16384: 65 against 76); up to eight they
// gain more than they lose (8 x 20480 x 16384 63 us against 83, 1 x 262144 x 4096 185 against 332, but 8 x 20480 x 4096 with
// zero points 34 against 31).
constexpr int kBlockSmem = 227 * 1024;
bool small_batch(int T, int K)
{
    const int cluster = T > 8 ? 4 : 8, chunks = (K + xs::kSwChunk - 1) / xs::kSwChunk;
    return T <= xs::kSwTokens && xs::sw_smem_bytes(T, (chunks + cluster - 1) / cluster, 2) <= kBlockSmem;
}

bool small_mlp(const XsMoeW4 *gu, const XsMoeW4 *dn, int T)
{
    return small_batch(T, gu->cols) && small_batch(T, dn->cols);
}

// Scratch of the tensor-core kernel: tokens and scales in f16, zero points, factors; of an MLP also its gated product.
struct TcScratch {
    size_t x16 = 0, h16 = 0, token = 0, h = 0, scales[2] = {}, zeros[2] = {}, row[2] = {}, bytes = 0;
};

int groups_pitch(const XsMoeW4 *w)
{
    return (w->cols / w->group + 7) / 8 * 8;
}

// Tokens whose gated product is in memory as f32 at one time: 512 MB of it, and all tokens up to there (8192 of 12288 columns are 403).
int gated_part(const XsMoeW4 *down, int T)
{
    constexpr size_t kBytes = size_t(512) << 20, kTile = 256;
    const size_t tokens = kBytes / (static_cast<size_t>(down->cols) * 4) / kTile * kTile, part = tokens < kTile ? kTile : tokens;
    return part < static_cast<size_t>(T) ? static_cast<int>(part) : T;
}

TcScratch plan_scratch(const XsMoeW4 *first, const XsMoeW4 *second, int T)
{
    TcScratch p;
    size_t at = kStatusBytes;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at = align_up(at + bytes, 256);
        return o;
    };
    const size_t x_bytes = static_cast<size_t>(T) * first->cols * 2, h16_bytes = second ? static_cast<size_t>(T) * second->cols * 2 : 0;
    const int part = second ? gated_part(second, T) : T;
    // the second product's tokens take the place of the first one's where those are done with
    p.x16 = p.h16 = take(part == T && h16_bytes > x_bytes ? h16_bytes : x_bytes);
    if (part < T)
        p.h16 = take(h16_bytes);
    p.token = take(static_cast<size_t>(T) * 4);
    if (second)
        p.h = take(static_cast<size_t>(part) * second->cols * 4);
    const XsMoeW4 *w[2] = {first, second};
    for (int i = 0; i < 2; i++) {
        if (!w[i])
            continue;
        const size_t n = static_cast<size_t>(w[i]->rows) * groups_pitch(w[i]);
        p.scales[i] = take(n * 2);
        p.zeros[i] = take(w[i]->zeros_dev ? n : 0);
        p.row[i] = take(static_cast<size_t>(w[i]->rows) * 4);
    }
    p.bytes = at;
    return p;
}

// Tokens (normed by `norm` where it is given) and the scales of up to two matrices.
int launch_prepare(const XsMoeW4 *first, const XsMoeW4 *second, const XsMoeBlockNorms *norm, const void *x, int T, uint8_t *ws, const TcScratch &p,
                   cudaStream_t st)
{
    DeviceInfo di;
    if (int rc = device_info(&di))
        return rc;
    xs::PrepareArgs a{};
    a.x = static_cast<const __nv_bfloat16 *>(x);
    if (norm) {
        a.norm_w = static_cast<const __nv_bfloat16 *>(norm->pre_weight_dev);
        a.eps = norm->eps;
        a.offset = norm->weight_offset;
    }
    a.x16 = reinterpret_cast<__half *>(ws + p.x16);
    a.factor = reinterpret_cast<float *>(ws + p.token);
    a.T = T;
    a.K = first->cols;
    const XsMoeW4 *w[2] = {first, second};
    int blocks = T;
    for (int i = 0; i < 2; i++) {
        if (!w[i])
            continue;
        xs::PrepareScales &m = a.m[i];
        m.scales = static_cast<const uint16_t *>(w[i]->scales_dev);
        m.zeros = w[i]->zeros_dev;
        m.scales16 = reinterpret_cast<uint16_t *>(ws + p.scales[i]);
        m.zeros8 = ws + p.zeros[i];
        m.factor = reinterpret_cast<float *>(ws + p.row[i]);
        m.rows = w[i]->rows;
        m.groups = w[i]->cols / w[i]->group;
        m.pitch = groups_pitch(w[i]);
        m.vec = m.groups % 8 == 0 && !misaligned(m.scales, 16) && !misaligned(m.zeros, 8);
        m.lanes = 1;
        while (m.lanes < 32 && m.lanes * 8 < m.groups)
            m.lanes *= 2;
        const int at_once = xs::kPrepThreads / m.lanes;
        // four rows a thread where there are enough of them for every SM (a product of 64 x 4096 x 32003: 41.5 us against 43.4; of 20 x
        // 4096 x 4096, which has too few: 12.4 against 11.7)
        m.per_block = at_once;
        if (m.rows > 8 * di.sms * at_once)
            m.per_block = 4 * at_once < xs::kPrepRows ? 4 * at_once : xs::kPrepRows;
        m.blocks = (m.rows + m.per_block - 1) / m.per_block;
        blocks += m.blocks;
    }
    XS_CUDA(launch_pdl(xs::w4_prepare_kernel, blocks, xs::kPrepThreads, 0, st, a));
    note_launch();
    return 0;
}

xs::TcOperands operands(const XsMoeW4 *w, const uint8_t *ws, const TcScratch &p, int i)
{
    xs::TcOperands o{};
    o.scales = reinterpret_cast<const uint16_t *>(ws + p.scales[i]);
    o.zeros = w->zeros_dev ? ws + p.zeros[i] : nullptr;
    o.row = reinterpret_cast<const float *>(ws + p.row[i]);
    o.token = reinterpret_cast<const float *>(ws + p.token);
    o.pitch = groups_pitch(w);
    return o;
}

size_t linear_bytes(const XsMoeW4 *w, int T)
{
    return small_batch(T, w->cols) ? kStatusBytes : plan_scratch(w, nullptr, T).bytes;
}

int run_linear(const XsMoeW4 *w, bool gated, int act, const void *x, int T, void *out, uint8_t *ws, cudaStream_t st)
{
    int32_t *status = reinterpret_cast<int32_t *>(ws);
    if (small_batch(T, w->cols))
        return run_small(w, gated, act, x, T, out, status, st);
    const TcScratch p = plan_scratch(w, nullptr, T);
    if (int rc = launch_prepare(w, nullptr, nullptr, x, T, ws, p, st))
        return rc;
    const xs::TcOperands ops = operands(w, ws, p, 0);
    __nv_bfloat16 *o = static_cast<__nv_bfloat16 *>(out);
    return gated ? launch_tc<true>(w, ws + p.x16, T, o, ops, act, status, st) : launch_tc<false>(w, ws + p.x16, T, o, ops, 0, status, st);
}

// The gated product and the down product share one scratch: behind the status block h alone, or what the tensor-core kernel needs.
size_t mlp_bytes(const XsMoeW4 *gu, const XsMoeW4 *dn, int T)
{
    if (small_mlp(gu, dn, T))
        return kStatusBytes + static_cast<size_t>(T) * (gu->rows / 2) * 4;
    return plan_scratch(gu, dn, T).bytes;
}

// norm: the rows of x are normed on the way to the tensor core (null for small batches, and where there is no norm).
// after_norm: a kernel of the same call made x, so the weights were complete before it began
int run_mlp(const XsMoeW4 *gu, const XsMoeW4 *dn, int32_t act, const XsMoeBlockNorms *norm, const void *x, int32_t T, void *out, uint8_t *ws, cudaStream_t st,
            bool after_norm = false)
{
    int32_t *status = reinterpret_cast<int32_t *>(ws);
    if (small_mlp(gu, dn, T)) {
        uint8_t *h = ws + kStatusBytes;
        if (int rc = launch_small<true, false>(gu, x, T, h, act, true, after_norm, status, st))
            return rc;
        return launch_small<false, true>(dn, h, T, out, 0, false, true, status, st);
    }
    const TcScratch p = plan_scratch(gu, dn, T);
    if (int rc = launch_prepare(gu, dn, norm, x, T, ws, p, st))
        return rc;
    float *h = reinterpret_cast<float *>(ws + p.h), *token = reinterpret_cast<float *>(ws + p.token);
    for (int t = 0, part = gated_part(dn, T); t < T; t += part) {
        const int n = part < T - t ? part : T - t;
        xs::TcOperands up = operands(gu, ws, p, 0);
        up.token += t;
        if (int rc = launch_tc<true>(gu, ws + p.x16 + static_cast<size_t>(t) * gu->cols * 2, n, h, up, act, status, st))
            return rc;
        __half *h16 = reinterpret_cast<__half *>(ws + p.h16) + static_cast<size_t>(t) * dn->cols;
        XS_CUDA(launch_pdl(xs::w4_rescale_kernel, n, xs::kRescaleThreads, 0, st, h, h16, token + t, dn->cols));
        note_launch();
    }
    return launch_tc<false>(dn, ws + p.h16, T, static_cast<__nv_bfloat16 *>(out), operands(dn, ws, p, 1), 0, status, st);
}

template <int GROUP, int ITER, bool ALIGNED>
int launch_norm_t(const xs::NormResidualArgs &a, int sms, cudaStream_t st)
{
    constexpr int threads = GROUP < 256 ? 256 : GROUP, per_block = threads / GROUP;
    const int blocks = (a.rows + per_block - 1) / per_block, slots = sms * (2048 / threads);
    XS_CUDA(launch_pdl(xs::norm_residual_kernel<GROUP, ITER, ALIGNED>, blocks < slots ? blocks : slots, threads, 0, st, a));
    note_launch();
    return 0;
}

template <bool ALIGNED>
int launch_norm_rows(const xs::NormResidualArgs &a, int sms, cudaStream_t st)
{
    const int pieces = (a.H + 7) / 8 + (ALIGNED ? 0 : 1); // an unaligned row may touch one more
    if (pieces <= 32)
        return launch_norm_t<32, 1, ALIGNED>(a, sms, st);
    if (pieces <= 64)
        return launch_norm_t<32, 2, ALIGNED>(a, sms, st);
    if (pieces <= 128)
        return launch_norm_t<128, 1, ALIGNED>(a, sms, st);
    // Few rows: as many threads as the row has pieces, since only latency counts; many rows: two to four pieces a thread, by what
    // leaves the fewest threads idle.  4096 columns, full gate: 64 rows 3.0 us against 3.4, 148 rows 3.5 against 3.8, 296 rows 4.5
    // either way, 1500 rows 14.0 against 13.1, 8192 rows 55.3 against 53.5 (6.3 TB/s).
    if (a.rows <= 2 * sms) {
        if (pieces <= 256)
            return launch_norm_t<256, 1, ALIGNED>(a, sms, st);
        if (pieces <= 512)
            return launch_norm_t<512, 1, ALIGNED>(a, sms, st);
        if (pieces <= 1024)
            return launch_norm_t<1024, 1, ALIGNED>(a, sms, st);
        return launch_norm_t<1024, 2, ALIGNED>(a, sms, st);
    }
    if (pieces <= 256)
        return launch_norm_t<128, 2, ALIGNED>(a, sms, st);
    if (pieces <= 384)
        return launch_norm_t<128, 3, ALIGNED>(a, sms, st);
    if (pieces <= 512)
        return launch_norm_t<256, 2, ALIGNED>(a, sms, st);
    if (pieces <= 768)
        return launch_norm_t<256, 3, ALIGNED>(a, sms, st);
    if (pieces <= 1024)
        return launch_norm_t<512, 2, ALIGNED>(a, sms, st);
    if (pieces <= 1536)
        return launch_norm_t<512, 3, ALIGNED>(a, sms, st);
    return launch_norm_t<512, 4, ALIGNED>(a, sms, st);
}

constexpr int kNormMaxHidden = 56 * 1024; // a row in shared memory as f32

int launch_norm_residual(const xs::NormResidualArgs &a, cudaStream_t st)
{
    DeviceInfo di;
    if (int rc = device_info(&di))
        return rc;
    uintptr_t low = 0;
    for (const void *p : {static_cast<const void *>(a.y), static_cast<const void *>(a.r), static_cast<const void *>(a.w_post), static_cast<const void *>(a.gate),
                          static_cast<const void *>(a.w_next), static_cast<const void *>(a.r_out), static_cast<const void *>(a.n_out)})
        low |= reinterpret_cast<uintptr_t>(p);
    if (low % 16 == 0 && a.H <= 16 * 1024 - 8)
        return a.H % 8 == 0 ? launch_norm_rows<true>(a, di.sms, st) : launch_norm_rows<false>(a, di.sms, st);
    if (low % 16 == 0 && a.H == 16 * 1024)
        return launch_norm_rows<true>(a, di.sms, st);
    const size_t smem = static_cast<size_t>(a.H) * 4;
    static SmemLimit limit;
    if (int rc = limit.set(xs::norm_residual_loop_kernel, kNormMaxHidden * 4))
        return rc;
    XS_CUDA(launch_pdl(xs::norm_residual_loop_kernel, a.rows, xs::kNrLoopThreads, smem, st, a));
    note_launch();
    return 0;
}

size_t gate_elems(int kind, size_t rows, size_t hidden)
{
    return kind == XS_MOE_GATE_CHANNEL ? hidden : kind == XS_MOE_GATE_ROW ? rows : kind == XS_MOE_GATE_FULL ? rows * hidden : 0;
}

int check_norm_shape(int gate_kind, const void *gate, int32_t rows, int32_t hidden)
{
    if (gate_kind < XS_MOE_GATE_NONE || gate_kind > XS_MOE_GATE_FULL)
        return fail(XS_MOE_ERR_INVALID_ARG, "unknown gate kind");
    if (rows < 0 || hidden <= 0)
        return fail(XS_MOE_ERR_INVALID_ARG, "shape mismatch: non-positive dimension");
    // a gate without elements (no rows) has no address
    if (gate ? gate_kind == XS_MOE_GATE_NONE : gate_elems(gate_kind, rows, hidden) != 0)
        return fail(XS_MOE_ERR_INVALID_ARG, "gate and gate kind disagree");
    if (rows > kMaxDim)
        return fail(XS_MOE_ERR_UNSUPPORTED, "rows must be at most 2^30");
    if (hidden > kNormMaxHidden)
        return fail(XS_MOE_ERR_UNSUPPORTED, "hidden must be at most %d", kNormMaxHidden);
    return 0;
}

int check_norm(const XsMoeNormResidual *a)
{
    if (!a)
        return fail(XS_MOE_ERR_INVALID_ARG, "arguments are null");
    if (a->reserved[0] || a->reserved[1])
        return fail(XS_MOE_ERR_INVALID_ARG, "reserved fields must be zero");
    if (int rc = check_norm_shape(a->gate_kind, a->gate_dev, a->rows, a->hidden))
        return rc;
    if (a->rows == 0)
        return 0;
    if (!a->residual_dev)
        return fail(XS_MOE_ERR_INVALID_ARG, "null tensor pointer");
    if ((a->next_weight_dev != nullptr) != (a->next_out_dev != nullptr))
        return fail(XS_MOE_ERR_INVALID_ARG, "next weight and next output go together");
    if (a->y_dev ? !a->residual_out_dev : (a->residual_out_dev || a->post_weight_dev || a->gate_dev || !a->next_out_dev))
        return fail(XS_MOE_ERR_INVALID_ARG, "y and residual_out go together; without y there is only the next norm");
    const void *ptr[] = {a->y_dev, a->residual_dev, a->post_weight_dev, a->gate_dev, a->next_weight_dev, a->residual_out_dev, a->next_out_dev};
    const char *name[] = {"y", "residual", "post weight", "gate", "next weight", "residual_out", "next_out"};
    const size_t full = static_cast<size_t>(a->rows) * a->hidden, h = a->hidden;
    const size_t elems[] = {full, full, h, gate_elems(a->gate_kind, a->rows, a->hidden), h, full, full};
    int dev = 0;
    if (int rc = current_device(&dev))
        return rc;
    for (int i = 0; i < 7; i++) {
        if (!ptr[i])
            continue;
        if (misaligned(ptr[i], 2))
            return fail(XS_MOE_ERR_INVALID_ARG, "tensors must be 2-byte aligned");
        if (int rc = check_on_device(ptr[i], dev, name[i]))
            return rc;
    }
    for (int o = 5; o < 7; o++)
        for (int i = 0; i < 7; i++) {
            // every element of y and residual is read by the thread that writes it, before it does: the same address is fine
            const bool in_place = i < 2 && ptr[i] == ptr[o];
            if (i != o && !in_place && overlap(ptr[o], elems[o] * 2, ptr[i], elems[i] * 2))
                return fail(XS_MOE_ERR_INVALID_ARG, "%s overlaps %s", name[o], name[i]);
        }
    return 0;
}

int run_norm(const XsMoeNormResidual *a, cudaStream_t st)
{
    if (a->rows == 0)
        return 0;
    xs::NormResidualArgs k;
    k.y = static_cast<const __nv_bfloat16 *>(a->y_dev);
    k.r = static_cast<const __nv_bfloat16 *>(a->residual_dev);
    k.w_post = static_cast<const __nv_bfloat16 *>(a->post_weight_dev);
    k.gate = static_cast<const __nv_bfloat16 *>(a->gate_dev);
    k.w_next = static_cast<const __nv_bfloat16 *>(a->next_weight_dev);
    k.r_out = static_cast<__nv_bfloat16 *>(a->residual_out_dev);
    k.n_out = static_cast<__nv_bfloat16 *>(a->next_out_dev);
    k.gate_kind = a->gate_kind;
    k.rows = a->rows;
    k.H = a->hidden;
    k.eps = a->eps;
    k.c = a->residual_scale;
    k.offset = a->weight_offset;
    return launch_norm_residual(k, st);
}

int check_block_norms(const XsMoeBlockNorms *n, int32_t rows, int32_t hidden)
{
    if (!n)
        return fail(XS_MOE_ERR_INVALID_ARG, "norms are null");
    if (n->reserved[0] || n->reserved[1])
        return fail(XS_MOE_ERR_INVALID_ARG, "reserved fields must be zero");
    if (int rc = check_norm_shape(n->gate_kind, n->gate_dev, rows, hidden))
        return rc;
    if (!n->pre_weight_dev)
        return fail(XS_MOE_ERR_INVALID_ARG, "null tensor pointer");
    return 0;
}

int check_block_norms_data(const XsMoeBlockNorms *n, int dev)
{
    const void *ptr[] = {n->pre_weight_dev, n->post_weight_dev, n->gate_dev};
    const char *name[] = {"pre weight", "post weight", "gate"};
    for (int i = 0; i < 3; i++) {
        if (!ptr[i])
            continue;
        if (misaligned(ptr[i], 2))
            return fail(XS_MOE_ERR_INVALID_ARG, "tensors must be 2-byte aligned");
        if (int rc = check_on_device(ptr[i], dev, name[i]))
            return rc;
    }
    return 0;
}

// what the norms of a block write must not be what they read later
int check_block_overlap(const XsMoeBlockNorms *n, int32_t rows, int32_t hidden, const void *out, const void *ws, size_t ws_bytes)
{
    const size_t h = static_cast<size_t>(hidden) * 2, full = h * rows, g = gate_elems(n->gate_kind, rows, hidden) * 2;
    const void *ptr[] = {n->pre_weight_dev, n->post_weight_dev, n->gate_dev};
    const size_t len[] = {h, h, g};
    for (int i = 0; i < 3; i++)
        if (overlap(ptr[i], len[i], out, full) || overlap(ptr[i], len[i], ws, ws_bytes))
            return fail(XS_MOE_ERR_INVALID_ARG, "a norm weight or the gate overlaps out or the workspace");
    return 0;
}

XsMoeNormResidual pre_norm(const XsMoeBlockNorms *n, const void *x, void *xn, int32_t rows, int32_t hidden)
{
    XsMoeNormResidual a{};
    a.residual_dev = x;
    a.next_weight_dev = n->pre_weight_dev;
    a.next_out_dev = xn;
    a.rows = rows;
    a.hidden = hidden;
    a.eps = n->eps;
    a.residual_scale = 1.0f;
    a.weight_offset = n->weight_offset;
    return a;
}

XsMoeNormResidual block_tail(const XsMoeBlockNorms *n, const void *y, const void *x, void *out, int32_t rows, int32_t hidden)
{
    XsMoeNormResidual a{};
    a.y_dev = y;
    a.residual_dev = x;
    a.post_weight_dev = n->post_weight_dev;
    a.gate_dev = n->gate_dev;
    a.gate_kind = n->gate_kind;
    a.residual_out_dev = out;
    a.rows = rows;
    a.hidden = hidden;
    a.eps = n->eps;
    a.residual_scale = n->residual_scale;
    a.weight_offset = n->weight_offset;
    return a;
}

// the fail() string may allocate: an exception of the host library becomes a status like every other failure
template <typename F>
int guarded(F &&f) noexcept
{
    try {
        return f();
    } catch (...) {
        return XS_MOE_ERR_CUDA;
    }
}

} // namespace

extern "C" {

int xs_moe_linear_w4_workspace_bytes(const XsMoeW4 *w, int32_t tokens, size_t *bytes)
{
    return guarded([&]() -> int {
        if (int rc = check_w4_shape(w, tokens))
            return rc;
        if (!bytes)
            return fail(XS_MOE_ERR_INVALID_ARG, "null out-pointer");
        *bytes = linear_bytes(w, tokens);
        return 0;
    });
}

int xs_moe_linear_w4(const XsMoeW4 *w, const void *x, int32_t tokens, void *out, void *ws, size_t ws_bytes, void *stream)
{
    return guarded([&]() -> int {
        if (int rc = check_w4_shape(w, tokens))
            return rc;
        if (tokens == 0)
            return 0;
        const size_t need = linear_bytes(w, tokens);
        if (int rc = check_workspace(ws, ws_bytes, need))
            return rc;
        int dev = 0;
        if (int rc = current_device(&dev))
            return rc;
        const size_t n_out = static_cast<size_t>(tokens) * w->rows;
        if (int rc = check_w4_data(w, out, n_out, ws, need, dev))
            return rc;
        if (int rc = check_io(x, static_cast<size_t>(tokens) * w->cols, out, n_out, ws, need, dev))
            return rc;
        return run_linear(w, false, 0, x, tokens, out, static_cast<uint8_t *>(ws), static_cast<cudaStream_t>(stream));
    });
}

int xs_moe_gated_w4(const XsMoeW4 *gate_up, int32_t activation, const void *x, int32_t tokens, void *h, void *ws, size_t ws_bytes, void *stream)
{
    return guarded([&]() -> int {
        if (int rc = check_gated_shape(gate_up, activation, tokens))
            return rc;
        if (tokens == 0)
            return 0;
        const size_t need = linear_bytes(gate_up, tokens);
        if (int rc = check_workspace(ws, ws_bytes, need))
            return rc;
        int dev = 0;
        if (int rc = current_device(&dev))
            return rc;
        const size_t n_out = static_cast<size_t>(tokens) * (gate_up->rows / 2);
        if (int rc = check_w4_data(gate_up, h, n_out, ws, need, dev))
            return rc;
        if (int rc = check_io(x, static_cast<size_t>(tokens) * gate_up->cols, h, n_out, ws, need, dev))
            return rc;
        return run_linear(gate_up, true, activation, x, tokens, h, static_cast<uint8_t *>(ws), static_cast<cudaStream_t>(stream));
    });
}

int xs_moe_mlp_w4_workspace_bytes(const XsMoeW4 *gate_up, const XsMoeW4 *down, int32_t tokens, size_t *bytes)
{
    return guarded([&]() -> int {
        if (int rc = check_mlp_shape(gate_up, down, XS_MOE_SILU, tokens))
            return rc;
        if (!bytes)
            return fail(XS_MOE_ERR_INVALID_ARG, "null out-pointer");
        *bytes = mlp_bytes(gate_up, down, tokens);
        return 0;
    });
}

int xs_moe_mlp_w4(const XsMoeW4 *gate_up, const XsMoeW4 *down, int32_t activation, const void *x, int32_t tokens, void *out, void *ws,
                  size_t ws_bytes, void *stream)
{
    return guarded([&]() -> int {
        if (int rc = check_mlp_shape(gate_up, down, activation, tokens))
            return rc;
        if (tokens == 0)
            return 0;
        const size_t need = mlp_bytes(gate_up, down, tokens);
        if (int rc = check_workspace(ws, ws_bytes, need))
            return rc;
        int dev = 0;
        if (int rc = current_device(&dev))
            return rc;
        const size_t n = static_cast<size_t>(tokens) * gate_up->cols;
        for (const XsMoeW4 *w : {gate_up, down})
            if (int rc = check_w4_data(w, out, n, ws, need, dev))
                return rc;
        if (int rc = check_io(x, n, out, n, ws, need, dev))
            return rc;
        return run_mlp(gate_up, down, activation, nullptr, x, tokens, out, static_cast<uint8_t *>(ws), static_cast<cudaStream_t>(stream));
    });
}

int xs_moe_norm_residual(const XsMoeNormResidual *args, void *stream)
{
    return guarded([&]() -> int {
        if (int rc = check_norm(args))
            return rc;
        return run_norm(args, static_cast<cudaStream_t>(stream));
    });
}

int xs_moe_mlp_w4_block_workspace_bytes(const XsMoeW4 *gate_up, const XsMoeW4 *down, int32_t tokens, size_t *bytes)
{
    if (int rc = xs_moe_mlp_w4_workspace_bytes(gate_up, down, tokens, bytes))
        return rc;
    *bytes += 2 * bf16_bytes(tokens, gate_up->cols);
    return 0;
}

int xs_moe_mlp_w4_block(const XsMoeW4 *gate_up, const XsMoeW4 *down, int32_t activation, const XsMoeBlockNorms *norms, const void *x,
                        int32_t tokens, void *out, void *ws, size_t ws_bytes, void *stream)
{
    return guarded([&]() -> int {
        if (int rc = check_mlp_shape(gate_up, down, activation, tokens))
            return rc;
        const int32_t H = gate_up->cols;
        if (int rc = check_block_norms(norms, tokens, H))
            return rc;
        if (tokens == 0)
            return 0;
        int dev = 0;
        if (int rc = current_device(&dev))
            return rc;
        if (int rc = check_block_norms_data(norms, dev))
            return rc;
        const size_t inner = mlp_bytes(gate_up, down, tokens), row_bytes = bf16_bytes(tokens, H), need = inner + 2 * row_bytes;
        if (int rc = check_workspace(ws, ws_bytes, need))
            return rc;
        const size_t n = static_cast<size_t>(tokens) * H;
        for (const XsMoeW4 *w : {gate_up, down})
            if (int rc = check_w4_data(w, out, n, ws, need, dev))
                return rc;
        if (int rc = check_io(x, n, out, n, ws, need, dev, true))
            return rc;
        if (int rc = check_block_overlap(norms, tokens, H, out, ws, need))
            return rc;
        uint8_t *base = static_cast<uint8_t *>(ws), *xn = base + inner, *y = xn + row_bytes;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        // Larger batches are normed where their tokens are made ready for the tensor core.  Small ones are normed by a pass of their
        // own, during which the gated product already fetches its weights: 12.9 us for one token of 4096 x 2048, where norming in
        // every block of the product took 14.4.
        const bool small = small_mlp(gate_up, down, tokens);
        if (small) {
            const XsMoeNormResidual pre = pre_norm(norms, x, xn, tokens, H);
            if (int rc = run_norm(&pre, st))
                return rc;
        }
        if (int rc = run_mlp(gate_up, down, activation, small ? nullptr : norms, small ? xn : x, tokens, y, base, st, small))
            return rc;
        const XsMoeNormResidual tail = block_tail(norms, y, x, out, tokens, H);
        return run_norm(&tail, st);
    });
}

int xs_moe_normed_block_workspace_bytes(const XsMoeConfig *cfg, size_t *bytes)
{
    if (int rc = xs_moe_workspace_bytes(cfg, bytes))
        return rc;
    *bytes = align_up(*bytes, 256) + 2 * bf16_bytes(cfg->num_tokens, cfg->hidden);
    return 0;
}

int xs_moe_normed_block_forward(const XsMoeConfig *cfg, const XsMoeWeights *w, const XsMoeBlockNorms *norms, const void *x, void *out,
                                void *ws, size_t ws_bytes, void *stream)
{
    return guarded([&]() -> int {
        size_t fwd = 0;
        if (int rc = xs_moe_workspace_bytes(cfg, &fwd))
            return rc;
        const int32_t T = cfg->num_tokens, H = cfg->hidden;
        if (int rc = check_block_norms(norms, T, H))
            return rc;
        if (T == 0)
            return 0;
        int dev = 0;
        if (int rc = current_device(&dev))
            return rc;
        if (int rc = check_block_norms_data(norms, dev))
            return rc;
        const size_t row_bytes = bf16_bytes(T, H), inner = align_up(fwd, 256), need = inner + 2 * row_bytes;
        if (int rc = check_workspace(ws, ws_bytes, need))
            return rc;
        const size_t n = static_cast<size_t>(T) * H;
        if (int rc = check_io(x, n, out, n, ws, need, dev, true))
            return rc;
        if (int rc = check_block_overlap(norms, T, H, out, ws, need))
            return rc;
        uint8_t *xn = static_cast<uint8_t *>(ws) + inner, *y = xn + row_bytes;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (norms->weight_offset == 0.0f && !misaligned(norms->pre_weight_dev, 16)) {
            if (int rc = xs_moe_rmsnorm(x, norms->pre_weight_dev, xn, T, H, norms->eps, stream))
                return rc;
        } else {
            const XsMoeNormResidual pre = pre_norm(norms, x, xn, T, H);
            if (int rc = run_norm(&pre, st))
                return rc;
        }
        if (int rc = xs_moe_forward(cfg, w, xn, y, ws, inner, stream))
            return rc;
        const XsMoeNormResidual tail = block_tail(norms, y, x, out, T, H);
        return run_norm(&tail, st);
    });
}

} // extern "C"
