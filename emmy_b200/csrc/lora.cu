// Low-rank adapters of many requests at once, beside a shared projection:
//     out[t] = y[t] + scaling[l] * B_l (A_l x[t]),  l = ids[t];  out[t] = y[t] where ids[t] is not an adapter's number.
// A projection that holds several linears side by side (q, k and v; gate and up) has one A per linear: section s of the columns reads
// A_l[s], B_l is [N, R] over all of them.
//
// One launch up to 256 rows.  A unit is a block of at most 16 (64 above 256 rows) rows of one adapter; a cluster of CTAs works on it:
//   rows     which rows share an adapter is worked out by every CTA from the ids alone (up to 256 of them: a row's rank among the rows of
//            its adapter, the rows whose rank is a multiple of 16 open a block).  Above, group.cu lists the blocks first.
//   shrink   h = A_l x by mma.sync m16n8k16 (rows as M, ranks as N), K cut over all warps of the cluster: every byte of x and A_l is
//            read by one warp, straight into the fragment's registers (16 bytes a lane: a lane's eight K values are the K indices
//            {2j, 2j+1, 2j+8, 2j+9} of two steps, in both operands alike).  The warps' sums meet in shared memory in warp order, the
//            CTAs' in distributed shared memory in rank order: no atomics, no workspace.
//   expand   every CTA takes a share of the columns in groups of 32: rows as M, columns as N, R as K.  The columns of a group are dealt
//            to the four MMA tiles so that a lane ends with eight neighbouring ones: y is read and written 16 bytes at a time.
// h is kept in f32 and enters the second product as two 16-bit numbers, value and remainder (bf16: 16 bits of fraction, f16: 22, after
// the row is brought to the top of f16's range by a power of two): the result is rounded once, as it is stored.
// mma.sync and not tcgen05: a decode batch is bound by the bytes of A and B, a prompt by those of x and y.
#include "group.cuh"
#include "mma_sync.cuh"

namespace eq {

constexpr int kLoraThreads = 256;
constexpr int kLoraWarps = kLoraThreads / 32;
constexpr int kLoraSelfPlan = kLoraThreads;  // rows up to which a CTA works out the blocks itself, one row a thread
constexpr int kLoraMaxSections = 8;
constexpr int kLoraMaxRanks = 1024;          // S * R
constexpr int kLoraWideRanks = 256;          // S * R up to which blocks have 64 rows above kLoraSelfPlan rows
constexpr int kLoraMaxAdapters = kGroupMaxKeys;
constexpr int kLoraPass = 32;                // ranks of a shrink pass

struct LoraParams {
    const void* x;        // [T][K]
    const void* y;        // [T][N]
    const void* a;        // [L][S][R][K]
    const void* b;        // [L][N][R]
    const float* scaling; // [L]
    const int32_t* ids;   // [T]
    void* out;            // [T][N], may be y
    const GroupBlock* blocks;  // above kLoraSelfPlan rows
    const int32_t* n_blocks;
    const int32_t* rows;
    int T, K, N, R, S, L;
    int in_place;
    int h_stride;                       // 16-bit elements of a row of h
    int ends[kLoraMaxSections];         // columns before the end of section s
    int group_ends[kLoraMaxSections];   // 32-column groups before the end of section s
};

__device__ __forceinline__ void lora_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void lora_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t lora_cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t lora_cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ float lora_peer_load(const float* mine, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ int lora_adapter(const LoraParams& p, int t) {
    const int id = p.ids[t];
    return id >= 0 && id < p.L ? id : -1;
}

template <typename T, int MT>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_kernel(const __grid_constant__ LoraParams p) {
    constexpr int kRows = 16 * MT;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int32_t rows_s[kRows];
    __shared__ __align__(16) int32_t ids_s[MT == 1 ? kLoraSelfPlan : 4];
    __shared__ int32_t lead_s[kLoraWarps];
    __shared__ int32_t block_s[3];
    __shared__ float mul_s[kRows];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, j = lane & 3;
    const int ranks = p.S * p.R;
    const uint32_t cta = lora_cluster_rank(), ctas = lora_cluster_size();
    const int unit = blockIdx.x / ctas;

    asm volatile("griddepcontrol.wait;" ::: "memory");  // everything read below may come from the kernel before
    // ---- the unit's adapter and rows (the same for all CTAs of the cluster)
    int adapter = -1, count = 0;
    if (MT == 1 && !p.blocks) {
        int mine = -2, rank = 0;
        if (tid < p.T) mine = lora_adapter(p, tid);
        ids_s[tid] = mine;
        if (tid == 0) block_s[0] = -2;
        __syncthreads();
        for (int i = 0; i < (p.T & ~3); i += 4) {
            const int4 v = *reinterpret_cast<const int4*>(ids_s + i);
            rank += (v.x == mine && i < tid) + (v.y == mine && i + 1 < tid) + (v.z == mine && i + 2 < tid) + (v.w == mine && i + 3 < tid);
        }
        for (int i = p.T & ~3; i < p.T; ++i) rank += ids_s[i] == mine && i < tid;
        const bool leads = tid < p.T && rank % kRows == 0 && !(mine < 0 && p.in_place);
        const uint32_t leaders = __ballot_sync(0xFFFFFFFFu, leads);
        if (lane == 0) lead_s[warp] = __popc(leaders);
        __syncthreads();
        int before = __popc(leaders & ((1u << lane) - 1));
        for (int w = 0; w < warp; ++w) before += lead_s[w];
        if (leads && before == unit) {
            block_s[0] = mine;
            block_s[1] = rank;
        }
        __syncthreads();
        adapter = block_s[0];
        if (adapter == -2) return;  // the whole cluster: fewer blocks than the launch allowed for
        const int from = block_s[1];
        const bool in = mine == adapter && rank >= from && rank < from + kRows;
        if (in) rows_s[rank - from] = tid;
        count = __syncthreads_count(in);
    } else {
        if (unit >= *p.n_blocks) return;
        const GroupBlock blk = p.blocks[unit];
        adapter = blk.key;
        count = blk.count;
        if (tid < count) rows_s[tid] = p.rows[blk.first + tid];
        __syncthreads();
    }

    const T* yin = static_cast<const T*>(p.y);
    T* out = static_cast<T*>(p.out);
    if (adapter < 0) {  // no adapter: a copy
        const int vecs = p.N / 8;
        for (int r = 0; r < count; ++r) {
            const uint4* src = reinterpret_cast<const uint4*>(yin + static_cast<size_t>(rows_s[r]) * p.N);
            uint4* dst = reinterpret_cast<uint4*>(out + static_cast<size_t>(rows_s[r]) * p.N);
            for (int v = cta * kLoraThreads + tid; v < vecs; v += ctas * kLoraThreads) dst[v] = src[v];
        }
        return;
    }
    const int tiles_m = (count + 15) >> 4;

    // ---- shrink
    float* part = reinterpret_cast<float*>(smem);            // [kRows][ranks]: this CTA's share of K
    float* red = part + kRows * ranks;                       // [warps][kRows][kLoraPass]; the split h lies here afterwards
    const T* x = static_cast<const T*>(p.x);
    const T* a = static_cast<const T*>(p.a) + static_cast<size_t>(adapter) * ranks * p.K;
    const int chunks = (p.K + 31) / 32, slices = ctas * kLoraWarps, slice = cta * kLoraWarps + warp;
    const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * slice / slices), c1 = static_cast<int>(static_cast<int64_t>(chunks) * (slice + 1) / slices);
    const T* xr[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 16 * m + 8 * h + g;
            xr[m][h] = r < count ? x + static_cast<size_t>(rows_s[r]) * p.K : nullptr;
        }
    for (int col = 0; col < ranks; col += kLoraPass) {
        float acc[MT][4][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.f;
#pragma unroll (MT == 1 ? 2 : 1)
        for (int c = c0; c < c1; ++c) {
            const int k = 32 * c + 8 * j;
            const bool in = k < p.K;  // K is a multiple of 8
            uint4 wv[4], xv[MT][2];
#pragma unroll
            for (int n = 0; n < 4; ++n)
                wv[n] = in && col + 8 * n < ranks ? __ldg(reinterpret_cast<const uint4*>(a + static_cast<size_t>(col + 8 * n + g) * p.K + k)) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    xv[m][h] = in && xr[m][h] ? __ldg(reinterpret_cast<const uint4*>(xr[m][h] + k)) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if (m < tiles_m) {
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        mma_16816<T>(acc[m][n], xv[m][0].x, xv[m][1].x, xv[m][0].y, xv[m][1].y, wv[n].x, wv[n].y);
                        mma_16816<T>(acc[m][n], xv[m][0].z, xv[m][1].z, xv[m][0].w, xv[m][1].w, wv[n].z, wv[n].w);
                    }
                }
            }
        }
        float* mine = red + warp * kRows * kLoraPass;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<float2*>(mine + (16 * m + 8 * h + g) * kLoraPass + 8 * n + 2 * j) = make_float2(acc[m][n][2 * h], acc[m][n][2 * h + 1]);
        __syncthreads();
        const int width = min(kLoraPass, ranks - col);
        for (int i = tid; i < kRows * kLoraPass; i += kLoraThreads) {
            const int r = i / kLoraPass, n = i % kLoraPass;
            if (n >= width) continue;
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < kLoraWarps; ++w) s += red[w * kRows * kLoraPass + i];
            part[r * ranks + col + n] = s;
        }
        __syncthreads();
    }
    lora_cluster_arrive();
    lora_cluster_wait();

    // ---- h of the whole K, scaled and split; a warp takes a row
    T* hi_s = reinterpret_cast<T*>(red);
    T* lo_s = hi_s + kRows * p.h_stride;
    const float scaling = p.scaling[adapter];
    constexpr int kKeep = (MT == 1 ? kLoraMaxRanks : kLoraWideRanks) / 32;
    for (int r = warp; r < kRows; r += kLoraWarps) {
        float h[kKeep];
        float big = 0.f;
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const int n = lane + 32 * i;
            h[i] = 0.f;
            if (n < ranks) {
                for (uint32_t c = 0; c < ctas; ++c) h[i] += lora_peer_load(part + r * ranks + n, c);
                h[i] *= scaling;
                big = fmaxf(big, fabsf(h[i]));
            }
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, off));
        float up = 1.f, down = 1.f;  // powers of two that bring the row's largest value to [2^13, 2^14) in f16, and back
        if (std::is_same<T, __half>::value && big > 0.f && big < INFINITY) {
            const int e = min(13 - ilogbf(big), 120);
            up = ldexpf(1.f, e);
            down = ldexpf(1.f, -e);
        }
        if (lane == 0) mul_s[r] = down;
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const int n = lane + 32 * i;
            if (n < ranks) split16<T>(h[i] * up, hi_s[r * p.h_stride + n], lo_s[r * p.h_stride + n]);
        }
    }
    lora_cluster_arrive();  // this CTA is done with the others' shared memory
    __syncthreads();

    // ---- expand
    const T* b = static_cast<const T*>(p.b) + static_cast<size_t>(adapter) * p.N * p.R;
    const int groups = p.group_ends[p.S - 1];
    const int g0 = static_cast<int>(static_cast<int64_t>(groups) * cta / ctas), g1 = static_cast<int>(static_cast<int64_t>(groups) * (cta + 1) / ctas);
    for (int gi = g0 + warp; gi < g1; gi += kLoraWarps) {
        int s = 0;
        while (gi >= p.group_ends[s]) ++s;
        const int n0 = (s ? p.ends[s - 1] : 0) + 32 * (gi - (s ? p.group_ends[s - 1] : 0)), n_end = p.ends[s];
        const T* wrow[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int n = n0 + 8 * (g >> 1) + 2 * t + (g & 1);
            wrow[t] = n < n_end ? b + static_cast<size_t>(n) * p.R + 4 * j : nullptr;
        }
        float acc[MT][4][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[m][t][e] = 0.f;
        const T* h_row = hi_s + g * p.h_stride + s * p.R + 4 * j;
        const size_t lo_at = static_cast<size_t>(kRows) * p.h_stride;
#pragma unroll (MT == 1 ? 2 : 1)
        for (int k = 0; k < p.R; k += 16) {
            const bool in = k + 4 * j < p.R;  // R is a multiple of 8
            uint2 wv[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) wv[t] = in && wrow[t] ? __ldg(reinterpret_cast<const uint2*>(wrow[t] + k)) : make_uint2(0, 0);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if (m < tiles_m) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const T* at = h_row + 16 * m * p.h_stride + k + half * lo_at;
                        uint2 top = make_uint2(0, 0), bottom = make_uint2(0, 0);
                        if (in) {
                            top = *reinterpret_cast<const uint2*>(at);
                            bottom = *reinterpret_cast<const uint2*>(at + 8 * p.h_stride);
                        }
#pragma unroll
                        for (int t = 0; t < 4; ++t) mma_16816<T>(acc[m][t], top.x, bottom.x, top.y, bottom.y, wv[t].x, wv[t].y);
                    }
                }
            }
        }
        const int n = n0 + 8 * j;
        if (n < n_end) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = 16 * m + 8 * h + g;
                    if (r < count) {
                        const size_t at = static_cast<size_t>(rows_s[r]) * p.N + n;
                        const float mul = mul_s[r];
                        uint4 v = *reinterpret_cast<const uint4*>(yin + at);
                        T* e = reinterpret_cast<T*>(&v);
#pragma unroll
                        for (int t = 0; t < 4; ++t)
#pragma unroll
                            for (int i = 0; i < 2; ++i) e[2 * t + i] = from_float<T>(fmaf(acc[m][t][2 * h + i], mul, to_float(e[2 * t + i])));
                        *reinterpret_cast<uint4*>(out + at) = v;
                    }
                }
        }
    }
    lora_cluster_wait();  // no CTA leaves while another may read its sums
}

template <typename T, int MT>
static int lora_launch(const LoraParams& p, int64_t units, cudaStream_t stream) {
    auto kernel = lora_kernel<T, MT>;
    constexpr int kRows = 16 * MT;
    const int ranks = p.S * p.R;
    const size_t red = static_cast<size_t>(kLoraWarps) * kRows * kLoraPass * sizeof(float);
    const size_t split = 2 * static_cast<size_t>(kRows) * p.h_stride * 2;
    const size_t smem = static_cast<size_t>(kRows) * ranks * sizeof(float) + (red > split ? red : split);
    static bool configured[64] = {};
    int dev = 0;
    EQ_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        EQ_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    int ctas = 8;
    while (ctas > 1 && units * ctas > 2 * sm_count()) ctas /= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(units * ctas));
    cfg.blockDim = dim3(kLoraThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    EQ_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, p));
    return EQ_OK;
}

static size_t lora_align(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace eq

using namespace eq;

extern "C" size_t eq_lora_workspace_bytes(int64_t T, int64_t L) {
    if (T <= kLoraSelfPlan || L <= 0) return 0;
    return lora_align(256 + static_cast<size_t>(group_max_blocks(T, L, 16)) * sizeof(GroupBlock)) + lora_align(static_cast<size_t>(T) * sizeof(int32_t));
}

extern "C" int eq_lora_add(const void* y, const void* x, const void* a, const void* b, const float* scaling, const int32_t* adapter_ids, int64_t T, int64_t K,
                           int64_t N, int64_t R, int64_t L, int64_t S, const int64_t* section_widths, int act_dtype, void* out, void* workspace,
                           size_t workspace_bytes, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    EQ_REQUIRE(T >= 0 && K > 0 && N > 0 && R > 0 && L > 0 && S > 0, EQ_ERR_BAD_ARG, "eq_lora_add: bad extents T=%lld K=%lld N=%lld R=%lld L=%lld S=%lld", (long long)T,
               (long long)K, (long long)N, (long long)R, (long long)L, (long long)S);
    EQ_REQUIRE(act_dtype == EQ_F16 || act_dtype == EQ_BF16, EQ_ERR_BAD_ARG, "eq_lora_add: activations and adapters must be f16 or bf16");
    EQ_REQUIRE(S <= kLoraMaxSections, EQ_ERR_UNSUPPORTED, "eq_lora_add: at most %d sections, got %lld", kLoraMaxSections, (long long)S);
    EQ_REQUIRE(K % 8 == 0 && N % 8 == 0 && R % 8 == 0, EQ_ERR_UNSUPPORTED, "eq_lora_add: K, N and the rank must be multiples of 8 (K=%lld N=%lld R=%lld)", (long long)K,
               (long long)N, (long long)R);
    EQ_REQUIRE(R <= kLoraMaxRanks && S * R <= kLoraMaxRanks && L <= kLoraMaxAdapters, EQ_ERR_UNSUPPORTED, "eq_lora_add: sections x rank up to %d and %d adapters, got %lld x %lld and %lld",
               kLoraMaxRanks, kLoraMaxAdapters, (long long)S, (long long)R, (long long)L);
    EQ_REQUIRE(T < (int64_t(1) << 31) / 64 && K < (int64_t(1) << 28) && N < (int64_t(1) << 28), EQ_ERR_UNSUPPORTED, "eq_lora_add: extents too large");
    LoraParams p = {};
    int64_t end = 0, groups = 0;
    for (int64_t s = 0; s < S; ++s) {
        const int64_t width = section_widths ? section_widths[s] : (S == 1 ? N : 0);
        EQ_REQUIRE(width > 0 && width % 8 == 0 && width <= N - end, EQ_ERR_BAD_ARG, "eq_lora_add: section %lld has %lld columns: positive multiples of 8 that add up to N", (long long)s,
                   (long long)width);
        end += width;
        groups += ceil_div(width, 32);
        p.ends[s] = static_cast<int>(end);
        p.group_ends[s] = static_cast<int>(groups);
    }
    EQ_REQUIRE(end == N, EQ_ERR_BAD_ARG, "eq_lora_add: the sections hold %lld of %lld columns", (long long)end, (long long)N);
    if (T == 0) return EQ_OK;
    EQ_REQUIRE(y && x && a && b && scaling && adapter_ids && out, EQ_ERR_BAD_ARG, "eq_lora_add: null pointer");
    EQ_REQUIRE(aligned(y, 16) && aligned(x, 16) && aligned(a, 16) && aligned(b, 16) && aligned(out, 16), EQ_ERR_BAD_ALIGN,
               "eq_lora_add: activations and adapters must be 16-byte aligned");
    EQ_REQUIRE(aligned(scaling, 4) && aligned(adapter_ids, 4), EQ_ERR_BAD_ALIGN, "eq_lora_add: scaling and adapter_ids must be 4-byte aligned");
    const size_t need = eq_lora_workspace_bytes(T, L);
    EQ_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), EQ_ERR_WORKSPACE,
               "eq_lora_add: workspace of %zu bytes (256-byte aligned) needed, %zu given", need, workspace_bytes);
    p.x = x;
    p.y = y;
    p.a = a;
    p.b = b;
    p.scaling = scaling;
    p.ids = adapter_ids;
    p.out = out;
    p.T = static_cast<int>(T);
    p.K = static_cast<int>(K);
    p.N = static_cast<int>(N);
    p.R = static_cast<int>(R);
    p.S = static_cast<int>(S);
    p.L = static_cast<int>(L);
    p.in_place = out == y;
    p.h_stride = static_cast<int>(ceil_div(S * R, 64) * 64 + 16);  // rows 32 bytes apart modulo 128: a half-warp's 8-byte reads meet every bank once
    if (T <= kLoraSelfPlan) {
        const int64_t units = group_max_blocks(T, L, 16);
        return act_dtype == EQ_F16 ? lora_launch<__half, 1>(p, units, stream) : lora_launch<__nv_bfloat16, 1>(p, units, stream);
    }
    const int block_rows = S * R <= kLoraWideRanks ? 64 : 16;
    unsigned char* base = static_cast<unsigned char*>(workspace);
    int32_t* n_blocks = reinterpret_cast<int32_t*>(base);
    GroupBlock* blocks = reinterpret_cast<GroupBlock*>(base + 256);
    int32_t* rows = reinterpret_cast<int32_t*>(base + lora_align(256 + static_cast<size_t>(group_max_blocks(T, L, 16)) * sizeof(GroupBlock)));
    p.blocks = blocks;
    p.n_blocks = n_blocks;
    p.rows = rows;
    const int st = group_rows_launch(adapter_ids, p.T, p.L, !p.in_place, block_rows, blocks, n_blocks, rows, stream);
    if (st != EQ_OK) return st;
    const int64_t units = group_max_blocks(T, L, block_rows);
    if (block_rows == 16) return act_dtype == EQ_F16 ? lora_launch<__half, 1>(p, units, stream) : lora_launch<__nv_bfloat16, 1>(p, units, stream);
    return act_dtype == EQ_F16 ? lora_launch<__half, 4>(p, units, stream) : lora_launch<__nv_bfloat16, 4>(p, units, stream);
}
