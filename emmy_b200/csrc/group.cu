// The list of row blocks by key: see group.cuh.  One CTA counts, scans and places.  Every warp has a run of neighbouring rows and counters of its
// own in shared memory, so that the rows of a key stay in their order without atomics (which row shares a block with which decides how a
// kernel cuts its sums: an order that changes from call to call would change bits); threads of a warp with the same key add once.
#include "group.cuh"

namespace eq {

constexpr int kGroupWarps = 32;       // up to kGroupFew keys; kGroupManyWarps above: their counters have to fit shared memory
constexpr int kGroupFew = 1279;
constexpr int kGroupManyWarps = 8;

// Exclusive scan over all threads of one value each.  Two barriers.
__device__ __forceinline__ int group_scan(int v, int32_t* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, sum, d);
        if (lane >= d) sum += up;
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    int others = lane < warp ? warp_sums[lane] : 0;  // (32 warps at most)
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) others += __shfl_xor_sync(0xFFFFFFFFu, others, d);
    __syncthreads();
    return others + sum - v;
}

__global__ void __launch_bounds__(32 * kGroupWarps) group_rows_kernel(const int32_t* __restrict__ ids, int T, int keys, int keep_rest, int block_shift, int cut,
                                                                      GroupBlock* __restrict__ blocks, int32_t* __restrict__ n_blocks, int32_t* rows,
                                                                      int* __restrict__ status) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ int32_t counts[];  // [warps][keys + 1] rows, then where the warp's next row of the key goes; four lists of keys + 1
    __shared__ int32_t warp_sums[kGroupWarps];
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5, kinds = keys + 1;
    for (int i = tid; i < warps * kinds; i += threads) counts[i] = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int run = (T + 32 * warps - 1) / (32 * warps) * 32;  // rows of a warp
    const int t0 = min(static_cast<int64_t>(run) * warp, static_cast<int64_t>(T)), t1 = min(t0 + run, T);
    int32_t* mine = counts + warp * kinds;
    int32_t *kind_rows = counts + warps * kinds, *kind_first = kind_rows + kinds, *kind_head = kind_first + kinds, *kind_block = kind_head + kinds;
    constexpr int kAhead = 8;  // ids in flight; where a warp has no more, they are read and matched once
    int kind[kAhead];
    uint32_t same[kAhead];  // the lanes of the same kind
    auto kinds_of = [&](int t) {
        int id[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) id[a] = t + 32 * a + lane < t1 ? ids[t + 32 * a + lane] : -1;
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            kind[a] = id[a] >= 0 && id[a] < keys ? id[a] : keep_rest && t + 32 * a + lane < t1 ? keys : -1;
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (t + 32 * a < t1) same[a] = __match_any_sync(0xFFFFFFFFu, kind[a]);
    };
    for (int t = t0; t < t1; t += 32 * kAhead) {
        kinds_of(t);
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (t + 32 * a >= t1) break;
            if (kind[a] >= 0 && __ffs(same[a]) - 1 == lane) mine[kind[a]] += __popc(same[a]);
            __syncwarp();
        }
    }
    __syncthreads();
    // where every kind and every warp's part of it begins; `per` neighbouring kinds a thread
    const int per = (kinds + threads - 1) / threads, from = min(tid * per, kinds), to = min(from + per, kinds);
    int sum = 0;
    for (int i = from; i < to; ++i) {
        int c = 0;
#pragma unroll 8
        for (int w = 0; w < warps; ++w) c += counts[w * kinds + i];
        kind_rows[i] = c;
        sum += c;
    }
    int at = group_scan(sum, warp_sums);
    for (int i = from; i < to; ++i) {
        kind_first[i] = at;
        kind_head[i] = 0;
#pragma unroll 8
        for (int w = 0; w < warps; ++w) {
            const int here = counts[w * kinds + i];
            counts[w * kinds + i] = at;
            at += here;
        }
    }
    __syncthreads();
    for (int t = t0; t < t1; t += 32 * kAhead) {
        if (run > 32 * kAhead) kinds_of(t);
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (t + 32 * a >= t1) break;
            if (kind[a] >= 0) rows[mine[kind[a]] + __popc(same[a] & ((1u << lane) - 1))] = t + 32 * a + lane;
            __syncwarp();
            if (kind[a] >= 0 && __ffs(same[a]) - 1 == lane) mine[kind[a]] += __popc(same[a]);
            __syncwarp();
        }
    }
    __syncthreads();
    if (cut) {
        // a warp a kind: from which of its rows on they are neighbours up to the last.  Where a row is, all behind it are: 32 places are asked at a time.
        for (int i = warp; i < kinds; i += warps) {
            const int c = kind_rows[i];
            if (c <= kGroupRun) continue;
            const int32_t* mine_rows = rows + kind_first[i];
            const int last = mine_rows[c - 1];
            int lo = 0, hi = c - 1;  // hi is
            while (lo < hi) {
                const int place = lo + static_cast<int>(static_cast<int64_t>(hi - lo) * lane / 32);
                const uint32_t in_run = __ballot_sync(0xFFFFFFFFu, last - mine_rows[place] == c - 1 - place);
                if (in_run & 1u) {
                    hi = lo;
                } else {
                    const int first_in = in_run ? __ffs(in_run) - 1 : 32;
                    const int old_lo = lo, old_hi = hi;
                    lo = old_lo + static_cast<int>(static_cast<int64_t>(old_hi - old_lo) * (first_in - 1) / 32) + 1;
                    if (first_in < 32) hi = old_lo + static_cast<int>(static_cast<int64_t>(old_hi - old_lo) * first_in / 32);
                }
            }
            if (lane == 0) kind_head[i] = c - lo >= kGroupRun ? lo : 0;
        }
        __syncthreads();
    }
    const int block_rows = 1 << block_shift;
    auto blocks_of = [&](int n) { return (n + block_rows - 1) >> block_shift; };
    int bsum = 0;
    for (int i = from; i < to; ++i) bsum += blocks_of(kind_head[i]) + blocks_of(kind_rows[i] - kind_head[i]);
    int bat = group_scan(bsum, warp_sums);
    for (int i = from; i < to; ++i) {
        kind_block[i] = bat;
        bat += blocks_of(kind_head[i]) + blocks_of(kind_rows[i] - kind_head[i]);
    }
    if (tid == threads - 1) {
        *n_blocks = bat;
        if (status) *status = 0;
    }
    __syncthreads();
    constexpr int kListers = 8;  // lanes that list a kind's blocks: most kinds have a few, a prompt's adapter hundreds
    for (int i = tid / kListers; i < kinds; i += threads / kListers) {
        const int c = kind_rows[i], head = kind_head[i], first = kind_first[i], block = kind_block[i], heads = blocks_of(head);
        for (int b = tid % kListers; b < heads + blocks_of(c - head); b += kListers) {
            const int r = b < heads ? b << block_shift : head + ((b - heads) << block_shift);
            blocks[block + b].key = i < keys ? i : -1;
            blocks[block + b].first = first + r;
            blocks[block + b].count = min(block_rows, (b < heads ? head : c) - r);
        }
    }
}

int group_rows_launch(const int32_t* ids, int T, int keys, bool keep_rest, int block_rows, bool cut, GroupBlock* blocks, int32_t* n_blocks, int32_t* rows,
                      int* status, cudaStream_t stream) {
    constexpr int kMost = 208 * 1024;
    static_assert((kGroupFew + 1) * (kGroupWarps + 4) * 4 <= kMost && (kGroupMaxKeys + 1) * (kGroupManyWarps + 4) * 4 <= kMost, "the counters");
    int shift = 0;
    while ((1 << shift) < block_rows) ++shift;
    EQ_REQUIRE(keys <= kGroupMaxKeys, EQ_ERR_UNSUPPORTED, "at most %d keys", kGroupMaxKeys);
    EQ_CUDA_OK(cudaFuncSetAttribute(group_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    const int warps = keys <= kGroupFew ? kGroupWarps : kGroupManyWarps;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(32 * warps);
    cfg.dynamicSmemBytes = static_cast<size_t>(warps + 4) * (keys + 1) * sizeof(int32_t);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    EQ_CUDA_OK(cudaLaunchKernelEx(&cfg, group_rows_kernel, ids, T, keys, static_cast<int>(keep_rest), shift, static_cast<int>(cut), blocks, n_blocks, rows, status));
    return EQ_OK;
}

}  // namespace eq
