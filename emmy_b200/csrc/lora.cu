// Low-rank adapters of many requests at once, beside a shared projection:
//     out[t] = y[t] + scaling[l] * B_l (A_l x[t]),  l = ids[t];  out[t] = y[t] where ids[t] is not an adapter's number.
// A projection that holds several linears side by side (q, k and v; gate and up) has one A per linear: section s of the columns reads
// A_l[s], B_l is [N, R] over all of them.
//
// Up to 256 rows one launch, lora_rows_kernel.  A unit is a block of at most 16 rows of one adapter; a cluster of CTAs works on it:
//   rows     which rows share an adapter is worked out by every CTA from the ids alone (a row's rank among the rows of its adapter; the rows
//            whose rank is a multiple of 16 open a block).
//   shrink   h = A_l x by mma.sync m16n8k16 (rows as M, ranks as N), K cut over all warps of the cluster: every byte of x and A_l is
//            read by one warp, straight into the fragment's registers (16 bytes a lane: a lane's eight K values are the K indices
//            {2j, 2j+1, 2j+8, 2j+9} of two steps, in both operands alike).  The warps' sums meet in shared memory in warp order, the
//            CTAs' in distributed shared memory in rank order: no atomics, no workspace.
//   expand   every CTA takes a share of the columns in groups of 32: rows as M, columns as N, R as K.  The columns of a group are dealt
//            to the four MMA tiles so that a lane ends with eight neighbouring ones: y is read and written 16 bytes at a time.  The
//            next group's B and y are on their way while a group is multiplied, the first one's before the CTAs have met.
// Above, three: group.cu lists blocks of at most 128 rows, lora_shrink_kernel writes h, lora_expand_kernel adds B h to y in tiles of 128 rows x
// 128 columns.  Both products run on tcgen05: the rows of a block lie anywhere, so the threads gather them by cp.async into the swizzled tile that
// the MMA reads, one or two steps ahead; two CTAs an SM, so that the sums of one are turned and added while the other's copies land.
// h is kept in f32 and enters the second product as two 16-bit numbers, value and remainder (bf16: 16 bits of fraction, f16: 22, after
// the row is brought to the top of f16's range by a power of two): the result is rounded once, as it is stored.
// Up to 16 rows a block, mma.sync and not tcgen05: a decode batch is bound by the bytes of A and B and by latency, and fragments need no trip through
// shared or tensor memory.
#include "group.cuh"
#include "mma_sync.cuh"
#include "tc_common.cuh"

namespace eq {

constexpr int kLoraThreads = 256;
constexpr int kLoraWarps = kLoraThreads / 32;
constexpr int kLoraSelfPlan = kLoraThreads;  // rows up to which a CTA works out the blocks itself, one row a thread
constexpr int kLoraMaxSections = 8;
constexpr int kLoraMaxRanks = 1024;          // S * R
constexpr int kLoraWideRanks = 256;          // S * R up to which blocks have 128 rows above kLoraSelfPlan rows
constexpr int kLoraMaxAdapters = kGroupMaxKeys;
constexpr int kLoraPass = 32;                // ranks of a shrink pass
constexpr int kLoraRows = 128;               // of a block then
constexpr int kLoraTile = 128;               // columns of an expand tile
constexpr int kLoraStages = 3;               // of the shrink
constexpr int kLoraSub = 128 * 128;          // bytes of 128 rows x 64 elements
constexpr int kLoraTurn = 32 * 36 * 4;       // a warp's 32 x 32 sums, rows 144 bytes apart
constexpr int kLoraRun = 4;                  // neighbouring tiles that a CTA takes at a time

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
    void* hi;             // [T][S R] h of the rows in their order of `rows`, value and remainder
    void* lo;
    float* mul;           // [T] what the products of a row are multiplied by
    int* status;          // a bounded wait ran out
    int T, K, N, R, S, L;
    int in_place;
    int h_stride;                       // 16-bit elements of a row of h in shared memory
    int ends[kLoraMaxSections];         // columns before the end of section s
    int group_ends[kLoraMaxSections];   // 32-column groups before the end of section s
    int tile_ends[kLoraMaxSections];    // kLoraTile-column tiles before the end of section s
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

// A_l x of the block's rows, this warp's slice of K, all warps' sums added: part[r][n] is this CTA's share.  Ends behind a barrier of the CTA.
template <typename T>
__device__ __forceinline__ void lora_shrink(const LoraParams& p, int adapter, int count, const int32_t* rows_s, float* part, float* red, int slice, int slices) {
    constexpr int kRows = 16;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, j = lane & 3;
    const int ranks = p.S * p.R;
    const T* x = static_cast<const T*>(p.x);
    const T* a = static_cast<const T*>(p.a) + static_cast<size_t>(adapter) * ranks * p.K;
    const int chunks = (p.K + 31) / 32;
    const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * slice / slices), c1 = static_cast<int>(static_cast<int64_t>(chunks) * (slice + 1) / slices);
    const T* x0 = g < count ? x + static_cast<size_t>(rows_s[g]) * p.K : nullptr;
    const T* x1 = g + 8 < count ? x + static_cast<size_t>(rows_s[g + 8]) * p.K : nullptr;
    for (int col = 0; col < ranks; col += kLoraPass) {
        float acc[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll 4
        for (int c = c0; c < c1; ++c) {
            const int k = 32 * c + 8 * j;
            const bool in = k < p.K;  // K is a multiple of 8
            const uint4 zero = make_uint4(0, 0, 0, 0);
            uint4 wv[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) wv[n] = in && col + 8 * n < ranks ? __ldg(reinterpret_cast<const uint4*>(a + static_cast<size_t>(col + 8 * n + g) * p.K + k)) : zero;
            const uint4 top = in && x0 ? __ldg(reinterpret_cast<const uint4*>(x0 + k)) : zero, bottom = in && x1 ? __ldg(reinterpret_cast<const uint4*>(x1 + k)) : zero;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                mma_16816<T>(acc[n], top.x, bottom.x, top.y, bottom.y, wv[n].x, wv[n].y);
                mma_16816<T>(acc[n], top.z, bottom.z, top.w, bottom.w, wv[n].z, wv[n].w);
            }
        }
        constexpr int kPitch = kLoraPass + 8;  // rows a quarter of the banks apart
        float* mine = red + warp * kRows * kPitch;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) *reinterpret_cast<float2*>(mine + (8 * h + g) * kPitch + 8 * n + 2 * j) = make_float2(acc[n][2 * h], acc[n][2 * h + 1]);
        __syncthreads();
        const int width = min(kLoraPass, ranks - col);
        for (int i = tid; i < count * kLoraPass; i += kLoraThreads) {
            const int r = i / kLoraPass, n = i % kLoraPass;
            if (n >= width) continue;
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < kLoraWarps; ++w) s += red[(w * kRows + r) * kPitch + n];
            part[r * ranks + col + n] = s;
        }
        __syncthreads();
    }
}

// A row of h over the cluster's shares (`part`: the row in this CTA's), scaled, by one warp: put(n, value, remainder) for every rank; the row's
// factor is returned.
template <typename T, int RANKS, typename Put>
__device__ __forceinline__ float lora_join(const float* part, int ranks, uint32_t ctas, float scaling, Put&& put) {
    const int lane = threadIdx.x & 31;
    float h[RANKS / 32];
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < RANKS / 32; ++i) {
        const int n = lane + 32 * i;
        h[i] = 0.f;
        if (32 * i < ranks) {  // the whole warp
            const float* at = part + min(n, ranks - 1);
            float v[8];
#pragma unroll
            for (uint32_t c = 0; c < 8; ++c) v[c] = c < ctas ? lora_peer_load(at, c) : 0.f;
#pragma unroll
            for (int c = 0; c < 8; ++c) h[i] += v[c];
            h[i] = n < ranks ? h[i] * scaling : 0.f;
            big = fmaxf(big, fabsf(h[i]));
        }
    }
    float up = 1.f, down = 1.f;  // powers of two that bring the row's largest value to [2^13, 2^14) in f16, and back
    if (std::is_same<T, __half>::value) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, off));
        if (big > 0.f && big < INFINITY) {
            const int e = min(13 + 127 - static_cast<int>(__float_as_uint(big) >> 23), 120);
            up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        }
    }
#pragma unroll
    for (int i = 0; i < RANKS / 32; ++i) {
        const int n = lane + 32 * i;
        if (n < ranks) {
            T hi, lo;
            split16<T>(h[i] * up, hi, lo);
            put(n, hi, lo);
        }
    }
    return down;
}

// y + delta of eight neighbouring columns of a row: acc's columns as the four tiles of a group hold them (first of the lane's two rows, or second).
template <typename T>
__device__ __forceinline__ uint4 lora_add8(uint4 v, const float (&acc)[4][4], int second, float mul) {
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) e[2 * t + i] = from_float<T>(fmaf(second ? acc[t][2 + i] : acc[t][i], mul, to_float(e[2 * t + i])));
    return v;
}

// ------------------------------------------------------------------------------------------------ up to 256 rows (or more than 256 ranks): blocks of 16 rows
template <typename T>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_rows_kernel(const __grid_constant__ LoraParams p) {
    constexpr int kRows = 16;
    constexpr int kChunks = 2;  // of 32 ranks: what a lane asks for at a time
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int32_t rows_s[kRows];
    __shared__ __align__(16) int32_t ids_s[kLoraSelfPlan];
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
    if (!p.blocks) {
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
    const float scaling = __ldg(p.scaling + adapter);
    float* part = reinterpret_cast<float*>(smem);  // [kRows][ranks]: this CTA's share of K
    float* red = part + kRows * ranks;             // [warps][kRows][kLoraPass + 8]; the split h lies here afterwards
    lora_shrink<T>(p, adapter, count, rows_s, part, red, cta * kLoraWarps + warp, ctas * kLoraWarps);
    lora_cluster_arrive();

    // ---- expand: this warp's groups of 32 columns, each in steps of 64 ranks; a step's B and its group's y are asked for one step ahead
    const T* b = static_cast<const T*>(p.b) + static_cast<size_t>(adapter) * p.N * p.R;
    const int groups = p.group_ends[p.S - 1];
    const int g0 = static_cast<int>(static_cast<int64_t>(groups) * cta / ctas), g1 = static_cast<int>(static_cast<int64_t>(groups) * (cta + 1) / ctas);
    const bool has0 = g < count, has1 = g + 8 < count;
    const size_t y0 = static_cast<size_t>(rows_s[has0 ? g : 0]) * p.N, y1 = static_cast<size_t>(rows_s[has1 ? g + 8 : 0]) * p.N;
    struct Group {
        int section, first, end;  // columns
    };
    auto group = [&](int gi) {
        Group v;
        v.section = 0;
        while (gi >= p.group_ends[v.section]) ++v.section;
        const int s = v.section;
        v.first = (s ? p.ends[s - 1] : 0) + 32 * (gi - (s ? p.group_ends[s - 1] : 0));
        v.end = p.ends[s];
        return v;
    };
    uint4 next_w[4][kChunks], next_y[2];
    auto ask_w = [&](const Group& v, int k0) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int n = v.first + 8 * (g >> 1) + 2 * t + (g & 1);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int k = k0 + 32 * c + 8 * j;
                next_w[t][c] = n < v.end && k < p.R ? ld_stream_v4(b + static_cast<size_t>(n) * p.R + k) : make_uint4(0, 0, 0, 0);
            }
        }
    };
    auto ask_y = [&](const Group& v) {
        const int n = v.first + 8 * j;
        next_y[0] = has0 && n < v.end ? *reinterpret_cast<const uint4*>(yin + y0 + n) : make_uint4(0, 0, 0, 0);
        next_y[1] = has1 && n < v.end ? *reinterpret_cast<const uint4*>(yin + y1 + n) : make_uint4(0, 0, 0, 0);
    };
    int gi = g0 + warp;
    Group now = {}, ahead = {};
    if (gi < g1) {
        ahead = group(gi);
        ask_w(ahead, 0);
        ask_y(ahead);
    }

    // ---- h of the whole K, scaled and split; a warp takes a row
    lora_cluster_wait();
    T* hi_s = reinterpret_cast<T*>(red);
    T* lo_s = hi_s + kRows * p.h_stride;
    for (int r = warp; r < count; r += kLoraWarps) {
        auto put = [&](int n, T hi, T lo) {
            hi_s[r * p.h_stride + n] = hi;
            lo_s[r * p.h_stride + n] = lo;
        };
        float mul;
        if (ranks <= 128) mul = lora_join<T, 128>(part + r * ranks, ranks, ctas, scaling, put);
        else mul = lora_join<T, kLoraMaxRanks>(part + r * ranks, ranks, ctas, scaling, put);
        if (lane == 0) mul_s[r] = mul;
    }
    lora_cluster_arrive();  // this CTA is done with the others' shared memory
    __syncthreads();

    const float mul0 = mul_s[has0 ? g : 0], mul1 = mul_s[has1 ? g + 8 : 0];
    const int lo_at = kRows * p.h_stride;
    for (; gi < g1; gi += kLoraWarps) {
        now = ahead;
        float acc[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
        uint4 yv[2];
        const T* h_row = hi_s + g * p.h_stride + now.section * p.R + 8 * j;
        for (int k0 = 0; k0 < p.R; k0 += 32 * kChunks) {
            uint4 wv[4][kChunks];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int c = 0; c < kChunks; ++c) wv[t][c] = next_w[t][c];
            if (k0 == 0) {
                yv[0] = next_y[0];
                yv[1] = next_y[1];
            }
            if (k0 + 32 * kChunks < p.R) {
                ask_w(now, k0 + 32 * kChunks);
            } else if (gi + kLoraWarps < g1) {
                ahead = group(gi + kLoraWarps);
                ask_w(ahead, 0);
                ask_y(ahead);
            }
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int k = k0 + 32 * c;
                if (k >= p.R) break;
                const bool in = k + 8 * j < p.R;  // R is a multiple of 8
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint4 top = make_uint4(0, 0, 0, 0), bottom = make_uint4(0, 0, 0, 0);
                    if (in && has0) top = *reinterpret_cast<const uint4*>(h_row + k + half * lo_at);
                    if (in && has1) bottom = *reinterpret_cast<const uint4*>(h_row + k + half * lo_at + 8 * p.h_stride);
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        mma_16816<T>(acc[t], top.x, bottom.x, top.y, bottom.y, wv[t][c].x, wv[t][c].y);
                        mma_16816<T>(acc[t], top.z, bottom.z, top.w, bottom.w, wv[t][c].z, wv[t][c].w);
                    }
                }
            }
        }
        const int n = now.first + 8 * j;
        if (n < now.end) {
            if (has0) *reinterpret_cast<uint4*>(out + y0 + n) = lora_add8<T>(yv[0], acc, 0, mul0);
            if (has1) *reinterpret_cast<uint4*>(out + y1 + n) = lora_add8<T>(yv[1], acc, 1, mul1);
        }
    }
    lora_cluster_wait();  // no CTA leaves while another may read its sums
}

// ------------------------------------------------------------------------------------------------ more rows: blocks of 128, h through memory
// 16-byte chunk c of row r of a tile of 64-element rows, as the MMA's 128-byte swizzle has it.
__device__ __forceinline__ uint32_t lora_sw(int r, int c) { return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)); }
// 16 bytes to shared memory, zeros where `in` is false.
__device__ __forceinline__ void lora_copy(uint32_t to, const void* from, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void lora_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void lora_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Every thread waits for an MMA's commit.  One that does not come is reported; nothing is waited for after that.
__device__ __forceinline__ bool lora_mma_done(uint32_t bar, uint32_t parity, bool broken, int* status) {
    if (broken) return false;
    if (tc::mbar_wait(bar, parity)) return true;
    atomicExch(status, 1);
    return false;
}

template <typename T>
constexpr uint32_t lora_fmt() {
    return std::is_same<T, __half>::value ? 0u : 1u;
}

// h of a block: 128 rows x all ranks, K in steps of 64 cut over the cluster.
template <typename T>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_shrink_kernel(const __grid_constant__ LoraParams p) {
    extern __shared__ __align__(128) unsigned char smem_raw[];
    __shared__ int32_t rows_s[kLoraRows];
    __shared__ __align__(8) uint64_t bars[kLoraStages];
    __shared__ uint32_t tmem_slot;
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ranks = p.S * p.R, n_mma = (ranks + 15) & ~15;
    const uint32_t cta = lora_cluster_rank(), ctas = lora_cluster_size();
    const int unit = blockIdx.x / ctas;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (unit >= *p.n_blocks) return;
    const GroupBlock blk = p.blocks[unit];
    if (blk.key < 0) return;
    uint32_t cols = 32;
    while (cols < static_cast<uint32_t>(n_mma)) cols *= 2;
    if (tid == 0) {
        for (int i = 0; i < kLoraStages; ++i) tc::mbar_init(tc::smem_u32(bars + i), 1);
        tc::mbar_fence_init();
    }
    if (warp == 0) tc::tmem_alloc(tc::smem_u32(&tmem_slot), cols);
    if (tid < kLoraRows) rows_s[tid] = p.rows[blk.first + min(tid, blk.count - 1)];  // rows behind the last one repeat it: nobody reads their sums
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    // with the TMEM columns in hand: a dependent grid that took them first and then waited for this one would never give them back
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    const float scaling = __ldg(p.scaling + blk.key);
    const T* a = static_cast<const T*>(p.a) + static_cast<size_t>(blk.key) * ranks * p.K;
    const int all = (p.K + 63) / 64;
    const int s0 = static_cast<int>(static_cast<int64_t>(all) * cta / ctas), steps = static_cast<int>(static_cast<int64_t>(all) * (cta + 1) / ctas) - s0;
    const int stage_bytes = kLoraSub + ((n_mma * 128 + 1023) & ~1023);
    const uint32_t base = tc::smem_u32(smem), bar0 = tc::smem_u32(bars);
    const int c = tid & 7, r0 = tid >> 3;
    const T* xr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) xr[i] = static_cast<const T*>(p.x) + static_cast<size_t>(rows_s[r0 + 32 * i]) * p.K;
    auto ask = [&](int step) {
        const uint32_t to = base + (step % kLoraStages) * stage_bytes;
        const int k = 64 * (s0 + step) + 8 * c;
        const bool in = k < p.K;
        const int from = in ? k : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) lora_copy(to + lora_sw(r0 + 32 * i, c), xr[i] + from, in);
        for (int r = r0; r < ranks; r += 32) lora_copy(to + kLoraSub + lora_sw(r, c), a + static_cast<size_t>(r) * p.K + from, in);
    };
    for (int i = 0; i < kLoraStages - 1; ++i) {
        if (i < steps) ask(i);
        lora_commit();
    }
    bool broken = false;
    const uint32_t idesc = tc::instr_desc(lora_fmt<T>(), lora_fmt<T>(), 128, static_cast<uint32_t>(n_mma));
    for (int step = 0; step < steps; ++step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kLoraStages - 2) : "memory");
        lora_proxy_fence();
        __syncthreads();
        if (tid == 0) {
            const uint32_t at = base + (step % kLoraStages) * stage_bytes;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
                tc::mma_f16(tmem, tc::smem_desc_k_sw128(at + ks * 32), tc::smem_desc_k_sw128(at + kLoraSub + ks * 32), idesc, step > 0 || ks > 0);
            tc::mma_commit(bar0 + 8 * (step % kLoraStages));
        }
        // the stage that the step before this one read is filled again
        if (step > 0 && !lora_mma_done(bar0 + 8 * ((step - 1) % kLoraStages), ((step - 1) / kLoraStages) & 1, broken, p.status)) broken = true;
        if (step + kLoraStages - 1 < steps) ask(step + kLoraStages - 1);
        lora_commit();
    }
    if (steps > 0 && !lora_mma_done(bar0 + 8 * ((steps - 1) % kLoraStages), ((steps - 1) / kLoraStages) & 1, broken, p.status)) broken = true;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    tc::fence_after_sync();
    // this CTA's share of the sums over the stages: [128][ranks + 4]
    float* part = reinterpret_cast<float*>(smem);
    const int pitch = ranks + 4;
    for (int c0 = 32 * (warp >> 2); c0 < ranks; c0 += 64) {
        const int row = 32 * (warp & 3) + lane;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (c0 + 16 * half >= ranks) continue;  // the whole warp
            uint32_t v[16];
            if (steps > 0) tc::tmem_ld_32x16(tmem + ((32u * (warp & 3)) << 16) + c0 + 16 * half, v);
            tc::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c0 + 16 * half + 4 * i < ranks)
                    *reinterpret_cast<uint4*>(part + row * pitch + c0 + 16 * half + 4 * i) =
                        steps > 0 ? make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]) : make_uint4(0, 0, 0, 0);
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 0) tc::tmem_dealloc(tmem, cols);
    lora_cluster_arrive();
    lora_cluster_wait();
    for (int r = cta * kLoraWarps + warp; r < blk.count; r += ctas * kLoraWarps) {
        T* hi = static_cast<T*>(p.hi) + static_cast<size_t>(blk.first + r) * ranks;
        T* lo = static_cast<T*>(p.lo) + static_cast<size_t>(blk.first + r) * ranks;
        const float mul = lora_join<T, kLoraWideRanks>(part + r * pitch, ranks, ctas, scaling, [&](int n, T vh, T vl) {
            hi[n] = vh;
            lo[n] = vl;
        });
        if (lane == 0) p.mul[blk.first + r] = mul;
    }
    lora_cluster_arrive();
    lora_cluster_wait();
}

// Tiles of 128 rows x 128 columns, steps of 64 ranks.  A CTA takes runs of neighbouring tiles; the runs are dealt over the CTAs, so that blocks
// of few rows and of many mix.
template <typename T>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_expand_kernel(const __grid_constant__ LoraParams p) {
    extern __shared__ __align__(128) unsigned char smem_raw[];
    __shared__ int32_t rows_s[kLoraRows];
    __shared__ float mul_s[kLoraRows];
    __shared__ __align__(8) uint64_t bars[2];
    __shared__ uint32_t tmem_slot;
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ranks = p.S * p.R, steps = (p.R + 63) / 64, vecs = p.R / 8;
    // [2 stages][128 columns x 64 ranks], h: [steps][value, remainder][128 rows x 64 ranks], [warps] sums being turned
    unsigned char* h_s = smem + 2 * kLoraSub;
    float* turn = reinterpret_cast<float*>(h_s + steps * 2 * kLoraSub + warp * kLoraTurn);
    if (tid == 0) {
        tc::mbar_init(tc::smem_u32(bars), 1);
        tc::mbar_init(tc::smem_u32(bars + 1), 1);
        tc::mbar_fence_init();
    }
    if (warp == 0) tc::tmem_alloc(tc::smem_u32(&tmem_slot), kLoraTile);
    // what no copy writes of the last sixteen ranks is zero, in both operands
    if (p.R % 16)
        for (int i = tid; i < (2 + 2 * steps) * kLoraSub / 16; i += kLoraThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // with the TMEM columns in hand
    const uint32_t tmem = tmem_slot, bar0 = tc::smem_u32(bars), b_at = tc::smem_u32(smem), h_at = b_at + 2 * kLoraSub;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int n_blocks = *p.n_blocks, tiles = p.tile_ends[p.S - 1];
    const int64_t units = static_cast<int64_t>(n_blocks) * tiles;
    const T* yin = static_cast<const T*>(p.y);
    T* out = static_cast<T*>(p.out);

    struct Tile {
        int block, section, first, end;
    };
    int64_t u = static_cast<int64_t>(blockIdx.x) * kLoraRun;  // this CTA's units: [(blockIdx.x + i gridDim.x) kLoraRun, + kLoraRun)
    auto locate = [&](int block, int t) {
        Tile v;
        v.block = block;
        v.section = 0;
        while (t >= p.tile_ends[v.section]) ++v.section;
        const int s = v.section;
        v.first = (s ? p.ends[s - 1] : 0) + kLoraTile * (t - (s ? p.tile_ends[s - 1] : 0));
        v.end = p.ends[s];
        return v;
    };
    auto tile = [&](int64_t at) {
        const int block = static_cast<int>(at / tiles);
        return locate(block, static_cast<int>(at - static_cast<int64_t>(block) * tiles));
    };
    const int c = tid & 7, r0 = tid >> 3;
    auto ask = [&](const Tile& v, int step, int stage) {
        const int key = p.blocks[v.block].key;
        if (key >= 0 && 8 * step + c < vecs) {
            const T* b = static_cast<const T*>(p.b) + (static_cast<size_t>(key) * p.N + v.first + r0) * p.R + 64 * step + 8 * c;
            const uint32_t to = b_at + stage * kLoraSub + lora_sw(r0, c);  // rows 32 apart have the same swizzle
#pragma unroll
            for (int i = 0; i < kLoraTile / 32; ++i)
                if (v.first + r0 + 32 * i < v.end) lora_copy(to + i * 32 * 128, b + static_cast<size_t>(32 * i) * p.R, true);
        }
        lora_commit();
    };
    const uint32_t idesc = tc::instr_desc(lora_fmt<T>(), lora_fmt<T>(), 128, kLoraTile);
    int n_step = 0;  // MMA steps issued so far
    bool broken = false;
    auto step_done = [&](int n) {
        if (!lora_mma_done(bar0 + 8 * (n & 1), (n >> 1) & 1, broken, p.status)) broken = true;
    };
    int held_block = -1, held_section = -1;
    Tile now = {};
    if (u < units) {
        now = tile(u);
        ask(now, 0, 0);
    }
    int stage = 0;
    const int quarter = warp & 3, row_in = lane >> 2, col_in = 64 * (warp >> 2) + 8 * (lane & 3);
    while (u < units) {
        int64_t u_next = u + 1;
        if (u_next % kLoraRun == 0) u_next += static_cast<int64_t>(gridDim.x - 1) * kLoraRun;
        const bool more = u_next < units;
        const Tile next = more ? tile(u_next) : now;
        const GroupBlock blk = p.blocks[now.block];
        if (held_block != now.block || held_section != now.section) {
            __syncthreads();  // everyone is done with the rows held so far; their MMAs are done
            if (tid < blk.count) rows_s[tid] = p.rows[blk.first + tid];
            if (blk.key >= 0) {
                if (tid < blk.count) mul_s[tid] = p.mul[blk.first + tid];
                for (int i = tid; i < blk.count * vecs; i += kLoraThreads) {
                    const int r = i / vecs, v = i - r * vecs;
                    const size_t from = static_cast<size_t>(blk.first + r) * ranks + now.section * p.R + 8 * v;
                    unsigned char* to = h_s + (v >> 3) * 2 * kLoraSub + lora_sw(r, v & 7);
                    *reinterpret_cast<uint4*>(to) = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.hi) + from));
                    *reinterpret_cast<uint4*>(to + kLoraSub) = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.lo) + from));
                }
            }
            held_block = now.block;
            held_section = now.section;
        }
        for (int step = 0; step < steps; ++step) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            lora_proxy_fence();
            tc::fence_before_sync();  // the sums of the tile before this one have been read
            __syncthreads();
            if (tid == 0 && blk.key >= 0) {
                tc::fence_after_sync();
                const int k16 = min(4, (p.R - 64 * step + 15) / 16);
                const uint32_t a_at = h_at + step * 2 * kLoraSub, w_at = b_at + stage * kLoraSub;
                for (int ks = 0; ks < k16; ++ks) {
                    const uint64_t w = tc::smem_desc_k_sw128(w_at + ks * 32);
                    tc::mma_f16(tmem, tc::smem_desc_k_sw128(a_at + ks * 32), w, idesc, step > 0 || ks > 0);
                    tc::mma_f16(tmem, tc::smem_desc_k_sw128(a_at + kLoraSub + ks * 32), w, idesc, true);
                }
                tc::mma_commit(bar0 + 8 * (n_step & 1));
            }
            // the other stage is filled again: the MMA that read it is done (it ended a tile, or is waited for here)
            if (step > 0 && blk.key >= 0) step_done(n_step - 1);
            if (blk.key >= 0) ++n_step;
            if (step + 1 < steps) ask(now, step + 1, stage ^ 1);
            else if (more) ask(next, 0, stage ^ 1);
            stage ^= 1;
        }
        // y of this thread's rows and columns, then the sums
        uint4 yv[4][2];
        size_t at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 32 * quarter + 8 * i + row_in;
            at[i] = 0;
            if (r < blk.count) {
                at[i] = static_cast<size_t>(rows_s[r]) * p.N + now.first + col_in;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (now.first + col_in + 32 * h < now.end) yv[i][h] = *reinterpret_cast<const uint4*>(yin + at[i] + 32 * h);
            }
        }
        if (blk.key >= 0) {
            step_done(n_step - 1);
            tc::fence_after_sync();
        }
        if (32 * quarter < blk.count) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (blk.key >= 0) {
                    uint32_t v[32];
                    tc::tmem_ld_32x32(tmem + ((32u * quarter) << 16) + 64 * (warp >> 2) + 32 * h, v);
                    tc::tmem_ld_wait();
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(turn + lane * 36 + 4 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    __syncwarp();
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 8 * i + row_in;
                    if (32 * quarter + r < blk.count && now.first + col_in + 32 * h < now.end) {
                        uint4 w = yv[i][h];
                        if (blk.key >= 0) {
                            const float mul = mul_s[32 * quarter + r];
                            const float4 d0 = *reinterpret_cast<const float4*>(turn + r * 36 + 8 * (lane & 3)), d1 = *reinterpret_cast<const float4*>(turn + r * 36 + 8 * (lane & 3) + 4);
                            const float d[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
                            T* e = reinterpret_cast<T*>(&w);
#pragma unroll
                            for (int q = 0; q < 8; ++q) e[q] = from_float<T>(fmaf(d[q], mul, to_float(e[q])));
                        }
                        *reinterpret_cast<uint4*>(out + at[i] + 32 * h) = w;
                    }
                }
            }
        }
        u = u_next;
        now = next;
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 0) tc::tmem_dealloc(tmem, kLoraTile);
}

static size_t lora_align(size_t v) { return (v + 255) / 256 * 256; }

// CTAs of a cluster: the largest of 8, 4, 2, 1 whose grid stays within `waves` rounds of two CTAs an SM.
static int lora_cluster(int64_t units, int waves) {
    int ctas = 8;
    while (ctas > 1 && units * ctas > 2 * waves * sm_count()) ctas /= 2;
    return ctas;
}

static int lora_launch(void (*kernel)(const LoraParams), const LoraParams& p, int64_t grid, int cluster, size_t smem, cudaStream_t stream) {
    EQ_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kLoraThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    EQ_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, p));
    return EQ_OK;
}

// Bytes of A's rows in a stage of the shrink.
static size_t lora_stage_rows(int ranks) { return (static_cast<size_t>((ranks + 15) & ~15) * 128 + 1023) & ~size_t(1023); }

template <typename T>
static int lora_forward(LoraParams p, int64_t T_, int64_t L, unsigned char* base, cudaStream_t stream) {
    const int ranks = p.S * p.R;
    const int block_rows = p.T > kLoraSelfPlan && ranks <= kLoraWideRanks ? kLoraRows : 16;
    const int64_t units = group_max_blocks(T_, L, block_rows);
    if (p.T > kLoraSelfPlan) {
        size_t o = 256;
        auto take = [&](size_t bytes) {
            void* at = base + o;
            o += lora_align(bytes);
            return at;
        };
        p.status = reinterpret_cast<int*>(base);
        int32_t* n_blocks = reinterpret_cast<int32_t*>(base) + 1;
        GroupBlock* blocks = static_cast<GroupBlock*>(take(static_cast<size_t>(units) * sizeof(GroupBlock)));
        int32_t* rows = static_cast<int32_t*>(take(static_cast<size_t>(T_) * 4));
        p.blocks = blocks;
        p.n_blocks = n_blocks;
        p.rows = rows;
        const int st = group_rows_launch(p.ids, p.T, p.L, !p.in_place, block_rows, blocks, n_blocks, rows, p.status, stream);
        if (st != EQ_OK) return st;
        if (block_rows == kLoraRows) {
            p.mul = static_cast<float*>(take(static_cast<size_t>(T_) * 4));
            p.hi = take(static_cast<size_t>(T_) * ranks * 2);
            p.lo = take(static_cast<size_t>(T_) * ranks * 2);
        }
    }
    if (block_rows == 16) {
        p.h_stride = (ranks + 63) / 64 * 64 + 32;  // rows 64 bytes apart modulo 128: the 16-byte reads of two rows meet every bank once
        const size_t red = static_cast<size_t>(kLoraWarps) * 16 * (kLoraPass + 8) * sizeof(float), split = 2 * static_cast<size_t>(16) * p.h_stride * 2;
        const int ctas = lora_cluster(units, 2);
        return lora_launch(lora_rows_kernel<T>, p, units * ctas, ctas, static_cast<size_t>(16) * ranks * sizeof(float) + (red > split ? red : split), stream);
    }
    const size_t stages = static_cast<size_t>(kLoraStages) * (kLoraSub + lora_stage_rows(ranks)), sums = static_cast<size_t>(kLoraRows) * (ranks + 4) * sizeof(float);
    const int ctas = lora_cluster(units, 1);
    const int st = lora_launch(lora_shrink_kernel<T>, p, units * ctas, ctas, 1024 + (stages > sums ? stages : sums), stream);
    if (st != EQ_OK) return st;
    const size_t smem = 1024 + static_cast<size_t>(2 + 2 * ((p.R + 63) / 64)) * kLoraSub + kLoraWarps * kLoraTurn;
    const int64_t runs = ceil_div(units * p.tile_ends[p.S - 1], kLoraRun), most = (smem <= 113 * 1024 ? 2 : 1) * sm_count();
    return lora_launch(lora_expand_kernel<T>, p, runs < most ? runs : most, 1, smem, stream);
}

}  // namespace eq

using namespace eq;

extern "C" size_t eq_lora_workspace_bytes(int64_t T, int64_t L, int64_t S, int64_t R) {
    if (T <= kLoraSelfPlan || L <= 0 || S <= 0 || R <= 0) return 0;
    const size_t lists = 256 + lora_align(static_cast<size_t>(group_max_blocks(T, L, 16)) * sizeof(GroupBlock)) + lora_align(static_cast<size_t>(T) * 4);
    if (S > kLoraWideRanks || R > kLoraWideRanks || S * R > kLoraWideRanks) return lists;
    return lists + lora_align(static_cast<size_t>(T) * 4) + 2 * lora_align(static_cast<size_t>(T) * S * R * 2);
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
    int64_t end = 0, groups = 0, tiles = 0;
    for (int64_t s = 0; s < S; ++s) {
        const int64_t width = section_widths ? section_widths[s] : (S == 1 ? N : 0);
        EQ_REQUIRE(width > 0 && width % 8 == 0 && width <= N - end, EQ_ERR_BAD_ARG, "eq_lora_add: section %lld has %lld columns: positive multiples of 8 that add up to N", (long long)s,
                   (long long)width);
        end += width;
        groups += ceil_div(width, 32);
        tiles += ceil_div(width, kLoraTile);
        p.ends[s] = static_cast<int>(end);
        p.group_ends[s] = static_cast<int>(groups);
        p.tile_ends[s] = static_cast<int>(tiles);
    }
    EQ_REQUIRE(end == N, EQ_ERR_BAD_ARG, "eq_lora_add: the sections hold %lld of %lld columns", (long long)end, (long long)N);
    if (T == 0) return EQ_OK;
    EQ_REQUIRE(y && x && a && b && scaling && adapter_ids && out, EQ_ERR_BAD_ARG, "eq_lora_add: null pointer");
    EQ_REQUIRE(aligned(y, 16) && aligned(x, 16) && aligned(a, 16) && aligned(b, 16) && aligned(out, 16), EQ_ERR_BAD_ALIGN,
               "eq_lora_add: activations and adapters must be 16-byte aligned");
    EQ_REQUIRE(aligned(scaling, 4) && aligned(adapter_ids, 4), EQ_ERR_BAD_ALIGN, "eq_lora_add: scaling and adapter_ids must be 4-byte aligned");
    const size_t need = eq_lora_workspace_bytes(T, L, S, R);
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
    unsigned char* base = static_cast<unsigned char*>(workspace);
    return act_dtype == EQ_F16 ? lora_forward<__half>(p, T, L, base, stream) : lora_forward<__nv_bfloat16>(p, T, L, base, stream);
}

extern "C" int eq_lora_status(const void* workspace, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    EQ_REQUIRE(workspace, EQ_ERR_BAD_ARG, "eq_lora_status: null workspace");
    int host = 0;
    EQ_CUDA_OK(cudaMemcpyAsync(&host, workspace, sizeof(int), cudaMemcpyDeviceToHost, stream));
    EQ_CUDA_OK(cudaStreamSynchronize(stream));
    EQ_REQUIRE(host == 0, EQ_ERR_TIMEOUT, "eq_lora_status: a bounded pipeline wait ran out (code %d)", host);
    return EQ_OK;
}
