// The list of row blocks by key: see group.cuh.  One CTA counts, scans and places.  Every warp has a run of neighbouring rows and counters of its
// own in shared memory, so that the rows of a key stay in their order without atomics (which row shares a block with which decides how a
// kernel cuts its sums: an order that changes from call to call would change bits); threads of a warp with the same key add once.
#include "group.cuh"

namespace eq {

constexpr int kGroupWarps = 32;       // up to kGroupFew keys; kGroupManyWarps above: their counters have to fit shared memory
constexpr int kGroupFew = 1279;
constexpr int kGroupManyWarps = 8;

__global__ void __launch_bounds__(32 * kGroupWarps) group_rows_kernel(const int32_t* __restrict__ ids, int T, int keys, int keep_rest, int block_rows,
                                                                      GroupBlock* __restrict__ blocks, int32_t* __restrict__ n_blocks,
                                                                      int32_t* __restrict__ rows, int* __restrict__ status) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ int32_t counts[];  // [warps][keys + 1] rows, then where the warp's next row of the key goes
    __shared__ int32_t warp_rows[kGroupWarps], warp_blocks[kGroupWarps];
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5, kinds = keys + 1;
    for (int i = tid; i < warps * kinds; i += threads) counts[i] = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int run = (T + 32 * warps - 1) / (32 * warps) * 32;  // rows of a warp
    const int t0 = min(static_cast<int64_t>(run) * warp, static_cast<int64_t>(T)), t1 = min(t0 + run, T);
    int32_t* mine = counts + warp * kinds;
    constexpr int kAhead = 4;  // ids in flight
    auto kind_of = [&](int t) {
        if (t >= t1) return -1;
        const int id = ids[t];
        return id >= 0 && id < keys ? id : keep_rest ? keys : -1;
    };
    for (int t = t0; t < t1; t += 32 * kAhead) {
        int kind[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) kind[a] = kind_of(t + 32 * a + lane);
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const uint32_t same = __match_any_sync(0xFFFFFFFFu, kind[a]);
            if (kind[a] >= 0 && __ffs(same) - 1 == lane) mine[kind[a]] += __popc(same);
            __syncwarp();
        }
    }
    __syncthreads();
    // exclusive scans over the kinds, `per` neighbouring ones a thread
    const int per = (kinds + threads - 1) / threads, from = min(tid * per, kinds), to = min(from + per, kinds);
    int sum = 0, bsum = 0;
    for (int i = from; i < to; ++i) {
        int c = 0;
        for (int w = 0; w < warps; ++w) c += counts[w * kinds + i];
        sum += c;
        bsum += (c + block_rows - 1) / block_rows;
    }
    int si = sum, bi = bsum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int su = __shfl_up_sync(0xFFFFFFFFu, si, d), bu = __shfl_up_sync(0xFFFFFFFFu, bi, d);
        if (lane >= d) {
            si += su;
            bi += bu;
        }
    }
    if (lane == 31) {
        warp_rows[warp] = si;
        warp_blocks[warp] = bi;
    }
    __syncthreads();
    int at = si - sum, bat = bi - bsum;
    for (int w = 0; w < warp; ++w) {
        at += warp_rows[w];
        bat += warp_blocks[w];
    }
    for (int i = from; i < to; ++i) {
        const int first = at;
        for (int w = 0; w < warps; ++w) {
            const int c = counts[w * kinds + i];
            counts[w * kinds + i] = at;
            at += c;
        }
        for (int r = first; r < at; r += block_rows, ++bat) {
            GroupBlock blk;
            blk.key = i < keys ? i : -1;
            blk.first = r;
            blk.count = min(block_rows, at - r);
            blocks[bat] = blk;
        }
    }
    if (tid == threads - 1) {
        *n_blocks = bat;
        if (status) *status = 0;
    }
    __syncthreads();
    for (int t = t0; t < t1; t += 32 * kAhead) {
        int kind[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) kind[a] = kind_of(t + 32 * a + lane);
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const uint32_t same = __match_any_sync(0xFFFFFFFFu, kind[a]);
            if (kind[a] >= 0) rows[mine[kind[a]] + __popc(same & ((1u << lane) - 1))] = t + 32 * a + lane;
            __syncwarp();
            if (kind[a] >= 0 && __ffs(same) - 1 == lane) mine[kind[a]] += __popc(same);
            __syncwarp();
        }
    }
}

int group_rows_launch(const int32_t* ids, int T, int keys, bool keep_rest, int block_rows, GroupBlock* blocks, int32_t* n_blocks, int32_t* rows,
                      int* status, cudaStream_t stream) {
    static_assert((kGroupFew + 1) * kGroupWarps * 4 <= 160 * 1024 && (kGroupMaxKeys + 1) * kGroupManyWarps * 4 <= 160 * 1024, "the counters");
    EQ_REQUIRE(keys <= kGroupMaxKeys, EQ_ERR_UNSUPPORTED, "at most %d keys", kGroupMaxKeys);
    EQ_CUDA_OK(cudaFuncSetAttribute(group_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    const int warps = keys <= kGroupFew ? kGroupWarps : kGroupManyWarps;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(32 * warps);
    cfg.dynamicSmemBytes = static_cast<size_t>(warps) * (keys + 1) * sizeof(int32_t);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    EQ_CUDA_OK(cudaLaunchKernelEx(&cfg, group_rows_kernel, ids, T, keys, static_cast<int>(keep_rest), block_rows, blocks, n_blocks, rows, status));
    return EQ_OK;
}

}  // namespace eq
