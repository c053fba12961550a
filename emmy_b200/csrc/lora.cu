// Low-rank adapters of many requests at once, beside a shared projection:
//     out[t] = y[t] + scaling[l] * B_l (A_l x[t]),  l = ids[t];  out[t] = y[t] where ids[t] is not an adapter's number.
// A projection that holds several linears side by side (q, k and v; gate and up) has one A per linear: section s of the columns reads
// A_l[s], B_l is [N, R] over all of them.
//
// Up to 256 rows, and up to 2048 where blocks have 16 rows (lora_block_rows), one launch, lora_rows_kernel.  A unit is a block of at most 16 rows of
// one adapter; a cluster of CTAs works on it:
//   rows     which rows share an adapter is worked out by every CTA from the ids alone (a row's rank among the rows of its adapter, by a match in its
//            warp and a table of the warps' counts; the rows whose rank is a multiple of 16 open a block).
//   shrink   h = A_l x by mma.sync m16n8k16 (rows as M, ranks as N), K cut over all warps of the cluster: every byte of x and A_l is
//            read by one warp, straight into the fragment's registers (16 bytes a lane: a lane's eight K values are the K indices
//            {2j, 2j+1, 2j+8, 2j+9} of two steps, in both operands alike).  The warps' sums meet in shared memory in warp order, the
//            CTAs' in distributed shared memory in rank order: no atomics, no workspace.
//   expand   every CTA takes a share of the columns in groups of 32: rows as M, columns as N, R as K.  The columns of a group are dealt
//            to the four MMA tiles so that a lane ends with eight neighbouring ones: y is read and written 16 bytes at a time.  The
//            next group's B and y are on their way while a group is multiplied, the first one's before the CTAs have met.
// Above, two, the first of them group.cu's list of the blocks (1999 rows of K=N=5120, rank 16: 26 us, 23 with the list made by every CTA); for larger
// calls three: blocks of at most 128 rows, lora_shrink_kernel writes h, lora_expand_kernel adds B h to y in tiles of 128 rows x 128 columns.  Both products
// run on tcgen05.  The shrink's threads gather the rows of a block, which lie anywhere, by cp.async into the swizzled tile that the MMA reads, three to six
// steps ahead; the expand's tiles come and go by TMA.
// The tiles hold up to 256 ranks in all and 128 of a section.  More stay in blocks of 16 rows at any size, whose A and B come from L2 again for each: 8192 rows,
// prompts of 3 adapters, K=4096, us (bytes at the rate of HBM): N = 4096 + 1024 + 1024 of rank 128 400 (43), N=4096 of rank 256 356 (33); 4096 + 1024 of rank
// 128, on the tiles, 112 (37).
// h is kept in f32 and enters the second product as two 16-bit numbers, value and remainder (bf16: 16 bits of fraction, f16: 22, after
// the row is brought to the top of f16's range by a power of two): the result is rounded once, as it is stored.
// Up to 16 rows a block, mma.sync and not tcgen05: a decode batch is bound by the bytes of A and B and by latency, and fragments need no trip through
// shared or tensor memory.
#include <math.h>

#include "group.cuh"
#include "mma_sync.cuh"
#include "tc_common.cuh"

namespace eq {

constexpr int kLoraThreads = 256;
constexpr int kLoraWarps = kLoraThreads / 32;
constexpr int kLoraSelfPlan = kLoraThreads;  // rows up to which a CTA works out the blocks itself, one row a thread, and needs no workspace
constexpr int kLoraSelfRows = 8 * kLoraThreads;  // and up to which it does so for blocks of 16 rows, eight rows a thread
constexpr int kLoraMaxSections = 8;
constexpr int kLoraMaxRanks = 1024;          // S * R
constexpr int kLoraWideRanks = 256;          // S * R, and
constexpr int kLoraWideRank = 128;           // R, up to which blocks have 128 rows above kLoraSelfPlan rows
constexpr int kLoraMaxAdapters = kGroupMaxKeys;
constexpr int kLoraPass = 32;                // ranks of a shrink pass
constexpr int kLoraRows = 128;               // of a block then
constexpr int kLoraTile = 128;               // columns of an expand tile
constexpr int kLoraStages = 6;               // of the shrink at most
constexpr int kLoraSub = 128 * 128;          // bytes of 128 rows x 64 elements

struct LoraParams {
    const void* x;        // [T][K]
    const void* y;        // [T][N]
    const void* a;        // [L][S][R][K]
    const void* b;        // [L][N][R]
    const float* scaling; // [L]
    const int32_t* ids;   // [T]
    void* out;            // [T][N], may be y
    GroupBlock* blocks;        // null: the CTAs work them out
    const int32_t* n_blocks;
    const int32_t* rows;
    void* hi;             // [T][S x R rounded up to 16] h of the rows in their order of `rows`, value and remainder
    void* lo;
    float* mul;           // [T] what the products of a row are multiplied by
    int* status;          // a bounded wait ran out
    int T, K, N, R, S, L;
    int in_place;
    int run;                            // neighbouring expand tiles that a CTA takes at a time
    int stages;                         // of the shrink: 3, or kLoraStages where they fit beside a second CTA
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

// A_l x of the block's rows, this warp's slice of K, all warps' sums added: part[r][n] is this CTA's share.  TILES x 8 ranks a pass, STEPS x 32 elements of K asked
// for at once; PASSES: there are several passes, the next one's first are asked for while the sums of one meet.  Ends behind a barrier of the CTA.
template <typename T, int TILES, int STEPS, bool PASSES>
__device__ __forceinline__ void lora_shrink(const LoraParams& p, int adapter, int count, const int32_t* rows_s, float* part, float* red, int slice, int slices) {
    constexpr int kRows = 16, kPass = 8 * TILES;
    static_assert(kPass <= kLoraPass, "the warps' sums");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, j = lane & 3;
    const int ranks = p.S * p.R;
    const T* x = static_cast<const T*>(p.x);
    const T* a = static_cast<const T*>(p.a) + static_cast<size_t>(adapter) * ranks * p.K;
    const int chunks = (p.K + 31) / 32;
    const int c0 = chunks * slice / slices, c1 = chunks * (slice + 1) / slices;  // (2^23 x 64 at most)
    const T* x0 = g < count ? x + static_cast<size_t>(rows_s[g]) * p.K : nullptr;
    const T* x1 = g + 8 < count ? x + static_cast<size_t>(rows_s[g + 8]) * p.K : nullptr;
    uint4 wv[STEPS][TILES], top[STEPS], bottom[STEPS];
    auto load = [&](int col, int c) {
        const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            const int k = 32 * (c + u) + 8 * j;
            const bool in = c + u < c1 && k < p.K;  // K is a multiple of 8
#pragma unroll
            for (int n = 0; n < TILES; ++n)
                wv[u][n] = in && col + 8 * n < ranks ? __ldg(reinterpret_cast<const uint4*>(a + static_cast<size_t>(col + 8 * n + g) * p.K + k)) : zero;
            top[u] = in && x0 ? __ldg(reinterpret_cast<const uint4*>(x0 + k)) : zero;
            bottom[u] = in && x1 ? __ldg(reinterpret_cast<const uint4*>(x1 + k)) : zero;
        }
    };
    if (PASSES) load(0, c0);
    for (int col = 0; col < ranks; col += kPass) {
        float acc[TILES][4];
#pragma unroll
        for (int n = 0; n < TILES; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
        for (int c = c0; c < c1; c += STEPS) {
            if (!PASSES) load(col, c);
#pragma unroll
            for (int u = 0; u < STEPS; ++u) {
                if (c + u >= c1) break;
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
                    mma_16816<T>(acc[n], top[u].x, bottom[u].x, top[u].y, bottom[u].y, wv[u][n].x, wv[u][n].y);
                    mma_16816<T>(acc[n], top[u].z, bottom[u].z, top[u].w, bottom[u].w, wv[u][n].z, wv[u][n].w);
                }
            }
            if (PASSES && c + STEPS < c1) load(col, c + STEPS);
        }
        if (PASSES && col + kPass < ranks) load(col + kPass, c0);
        constexpr int kPitch = kLoraPass + 8;  // rows a quarter of the banks apart
        float* mine = red + warp * kRows * kPitch;
#pragma unroll
        for (int n = 0; n < TILES; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) *reinterpret_cast<float2*>(mine + (8 * h + g) * kPitch + 8 * n + 2 * j) = make_float2(acc[n][2 * h], acc[n][2 * h + 1]);
        __syncthreads();
        const int width = min(kPass, ranks - col);
        for (int i = tid; i < count * kPass; i += kLoraThreads) {
            const int r = i / kPass, n = i % kPass;
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
            const float size = fabsf(h[i]);
            big = size < INFINITY ? fmaxf(big, size) : big;  // (an infinity in one section's sums is no reason to leave another's out of range)
        }
    }
    float up = 1.f, down = 1.f;  // powers of two that bring the row's largest finite value to [2^13, 2^14) in f16, and back
    if (std::is_same<T, __half>::value) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, off));
        if (big > 0.f) {
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

// Two neighbouring values plus v0 mul and v1 mul.
template <typename T>
__device__ __forceinline__ uint32_t lora_add2(uint32_t y, float v0, float v1, float mul) {
    if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&y));
        const __half2 h = __floats2half2_rn(fmaf(v0, mul, f.x), fmaf(v1, mul, f.y));
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(fmaf(v0, mul, __uint_as_float(y << 16)), fmaf(v1, mul, __uint_as_float(y & 0xFFFF0000u)));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
// y + delta of eight neighbouring columns of a row: acc's columns as the four tiles of a group hold them (first of the lane's two rows, or second).
template <typename T>
__device__ __forceinline__ uint4 lora_add8(uint4 v, const float (&acc)[4][4], int second, float mul) {
    const int at = 2 * second;
    return make_uint4(lora_add2<T>(v.x, acc[0][at], acc[0][at + 1], mul), lora_add2<T>(v.y, acc[1][at], acc[1][at + 1], mul),
                      lora_add2<T>(v.z, acc[2][at], acc[2][at + 1], mul), lora_add2<T>(v.w, acc[3][at], acc[3][at + 1], mul));
}

// ------------------------------------------------------------------------------------------------ blocks of 16 rows
// Bound by latency for few bytes: one row of K=N=4096, rank 16, takes 5.0 us a launch beside 0.04 us of bytes, 17 rows of K=14336 N=4096, rank 32, 7.9 us (0.8), and
// by how soon A's and B's bytes are asked for: 256 rows of 64 adapters, K=5120 N=34816, rank 64, 84 us for 396 MB, 4.7 TB/s.  With four warps a scheduler the
// instructions between two loads are part of that latency: 64-bit divisions of the shares and zeros for what nobody stores were a fifth of either time.
// kSmall: no more than sixteen ranks in all, half the fragments, so more of them are asked for at once.
// kChunks: of 32 ranks, what a lane asks for at a time; one where there are no more (K=14336 N=4096, rank 32, 17 rows 8.8 us against 10.2; three CTAs an
// SM then, of 80 registers, 10.5).
template <typename T, int kChunks, bool kSmall>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_rows_kernel(const __grid_constant__ LoraParams p) {
    constexpr int kRows = 16;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    static_assert(!kSmall || kChunks == 1, "");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int32_t rows_s[kRows];
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
    if (!p.blocks && p.T > kLoraSelfPlan) {
        // Every warp has a run of neighbouring rows and counts the kinds in it; the blocks lie in the order of their kinds, rows without an adapter last.
        if (blockIdx.x == 0 && tid == 0) *p.status = 0;
        uint4* counts = reinterpret_cast<uint4*>(smem);  // [L + 1] rows of each warp, 16 bits
        if (tid == 0) block_s[0] = -2;
        for (int i = tid; i <= p.L; i += kLoraThreads) counts[i] = make_uint4(0, 0, 0, 0);
        constexpr int kMine = kLoraSelfRows / kLoraThreads;
        const int steps = (p.T + kLoraThreads - 1) / kLoraThreads, t0 = 32 * steps * warp + lane;
        int kind[kMine], rank[kMine];
#pragma unroll
        for (int c = 0; c < kMine; ++c) {
            kind[c] = -1;
            if (c < steps && t0 + 32 * c < p.T) {
                const int id = lora_adapter(p, t0 + 32 * c);
                kind[c] = id >= 0 ? id : p.L;
            }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kMine; ++c) {
            if (c >= steps) break;
            const uint32_t same = __match_any_sync(0xFFFFFFFFu, kind[c]);
            uint16_t* mine = reinterpret_cast<uint16_t*>(counts + max(kind[c], 0)) + warp;
            const int before = kind[c] >= 0 ? *mine : 0;
            rank[c] = before + __popc(same & ((1u << lane) - 1));
            __syncwarp();
            if (kind[c] >= 0 && __ffs(same) - 1 == lane) *mine = static_cast<uint16_t>(before + __popc(same));
            __syncwarp();
        }
        __syncthreads();
        // rows of kind i in the first `warps` warps' runs
        auto rows_of = [&](int i, int warps) {
            const uint4 v = counts[i];
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            uint32_t sum = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) sum += (2 * q < warps ? w[q] & 0xFFFFu : 0u) + (2 * q + 1 < warps ? w[q] >> 16 : 0u);
            return static_cast<int>(sum);
        };
        const int kinds = p.in_place ? p.L : p.L + 1, per = (kinds + kLoraThreads - 1) / kLoraThreads, from_kind = min(tid * per, kinds), to_kind = min(from_kind + per, kinds);
        int blocks = 0;
        for (int i = from_kind; i < to_kind; ++i) blocks += (rows_of(i, kLoraWarps) + kRows - 1) / kRows;
        int at = blocks;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xFFFFFFFFu, at, d);
            if (lane >= d) at += up;
        }
        if (lane == 31) lead_s[warp] = at;
        __syncthreads();
        at -= blocks;
        for (int w = 0; w < warp; ++w) at += lead_s[w];
        if (at <= unit && unit < at + blocks) {
            for (int i = from_kind; i < to_kind; ++i) {
                const int n = rows_of(i, kLoraWarps), its = (n + kRows - 1) / kRows;
                if (unit < at + its) {
                    block_s[0] = i;
                    block_s[1] = kRows * (unit - at);
                    block_s[2] = min(kRows, n - block_s[1]);
                    break;
                }
                at += its;
            }
        }
        __syncthreads();
        const int target = block_s[0];
        if (target == -2) return;  // the whole cluster: fewer blocks than the launch allowed for
        const int first = block_s[1] - rows_of(target, warp);
#pragma unroll
        for (int c = 0; c < kMine; ++c)
            if (c < steps && kind[c] == target && rank[c] >= first && rank[c] < first + kRows) rows_s[rank[c] - first] = t0 + 32 * c;
        adapter = target < p.L ? target : -1;
        count = block_s[2];
        __syncthreads();
    } else if (!p.blocks) {
        // a row's rank: the rows of its kind ahead of it in its warp, and those that the warps before counted, a byte a warp
        const int mine = tid < p.T ? lora_adapter(p, tid) : -2;
        const uint32_t same = __match_any_sync(0xFFFFFFFFu, mine);
        int rank = __popc(same & ((1u << lane) - 1));
        if (tid == 0) block_s[0] = -2;
        if (p.T > 32) {
            uint2* counts = reinterpret_cast<uint2*>(smem);  // [L + 1]
            const int kind = mine >= 0 ? mine : p.L;
            for (int i = tid; i <= p.L; i += kLoraThreads) counts[i] = make_uint2(0, 0);
            __syncthreads();
            if (tid < p.T && rank == 0) reinterpret_cast<uint8_t*>(counts + kind)[warp] = static_cast<uint8_t>(__popc(same));
            __syncthreads();
            const uint2 others = counts[kind];
            const uint64_t ahead_of = ((static_cast<uint64_t>(others.y) << 32) | others.x) & ((uint64_t(1) << (8 * warp)) - 1);
            rank = static_cast<int>(__dp4a(static_cast<uint32_t>(ahead_of), 0x01010101u, __dp4a(static_cast<uint32_t>(ahead_of >> 32), 0x01010101u, static_cast<uint32_t>(rank))));
        }
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
    lora_shrink<T, kSmall ? 2 : 4, kSmall ? 5 : kChunks + 1, kChunks == 2>(p, adapter, count, rows_s, part, red, cta * kLoraWarps + warp, ctas * kLoraWarps);
    lora_cluster_arrive();

    // ---- expand: this warp's groups of 32 columns, each in steps of 64 ranks; a step's B and its group's y are asked for one step ahead
    const T* b = static_cast<const T*>(p.b) + static_cast<size_t>(adapter) * p.N * p.R;
    const int groups = p.group_ends[p.S - 1];
    const int g0 = groups * static_cast<int>(cta) / static_cast<int>(ctas), g1 = groups * static_cast<int>(cta + 1) / static_cast<int>(ctas);
    const bool has0 = g < count, has1 = g + 8 < count;
    const size_t y0 = static_cast<size_t>(rows_s[has0 ? g : 0]) * p.N, y1 = static_cast<size_t>(rows_s[has1 ? g + 8 : 0]) * p.N;
    struct Group {
        int section, first, end;  // columns
    };
    int section = 0, groups_before = 0, columns_before = 0, group_end = p.group_ends[0], column_end = p.ends[0];
    auto group = [&](int gi) {  // they ascend
        while (gi >= group_end) {
            groups_before = group_end;
            columns_before = column_end;
            ++section;
            group_end = p.group_ends[section];
            column_end = p.ends[section];
        }
        return Group{section, columns_before + 32 * (gi - groups_before), column_end};
    };
    // (with sixteen ranks a lane has four of them, eight bytes of B, and three groups are on their way)
    constexpr int kAhead = kSmall ? 3 : 1;
    uint4 next_w[4][kChunks], next_y[kAhead][2];
    uint2 next_s[kAhead][4] = {};  // (lanes without ranks keep the zeros; columns and rows that nobody stores keep what is there)
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
    const int n_s = 8 * (g >> 1) + (g & 1);
    const T* b_s = b + n_s * p.R + 4 * j;
    auto ask_s = [&](const Group& v, uint2 (&to)[4]) {
        const T* at = b_s + static_cast<size_t>(v.first) * p.R;
        const int left = 4 * j < p.R ? v.end - v.first - n_s : 0;
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (2 * t < left) to[t] = __ldg(reinterpret_cast<const uint2*>(at + 2 * t * p.R));
    };
    auto ask_y = [&](const Group& v, uint4 (&to)[2]) {
        const int n = v.first + 8 * j;
        if (has0 && n < v.end) to[0] = *reinterpret_cast<const uint4*>(yin + y0 + n);
        if (has1 && n < v.end) to[1] = *reinterpret_cast<const uint4*>(yin + y1 + n);
    };
    int gi = g0 + warp;
    Group ahead[kAhead] = {};
    if constexpr (kSmall) {
#pragma unroll
        for (int d = 0; d < kAhead; ++d)
            if (gi + d * kLoraWarps < g1) {
                ahead[d] = group(gi + d * kLoraWarps);
                ask_s(ahead[d], next_s[d]);
                ask_y(ahead[d], next_y[d]);
            }
    } else if (gi < g1) {
        ahead[0] = group(gi);
        ask_w(ahead[0], 0);
        ask_y(ahead[0], next_y[0]);
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
        if (kSmall) mul = lora_join<T, 32>(part + r * ranks, ranks, ctas, scaling, put);
        else if (ranks <= 128) mul = lora_join<T, 128>(part + r * ranks, ranks, ctas, scaling, put);
        else mul = lora_join<T, kChunks == 1 ? 32 * kLoraMaxSections : kLoraMaxRanks>(part + r * ranks, ranks, ctas, scaling, put);
        if (lane == 0) mul_s[r] = mul;
    }
    lora_cluster_arrive();  // this CTA is done with the others' shared memory
    __syncthreads();

    const float mul0 = mul_s[has0 ? g : 0], mul1 = mul_s[has1 ? g + 8 : 0];
    const int lo_at = kRows * p.h_stride;
    auto put = [&](const Group& v, const uint4 (&yv)[2], const float (&acc)[4][4]) {
        const int n = v.first + 8 * j;
        if (n < v.end) {
            if (has0) *reinterpret_cast<uint4*>(out + y0 + n) = lora_add8<T>(yv[0], acc, 0, mul0);
            if (has1) *reinterpret_cast<uint4*>(out + y1 + n) = lora_add8<T>(yv[1], acc, 1, mul1);
        }
    };
    if constexpr (kSmall) {
        uint2 h[2][2] = {};  // value and remainder, rows g and g + 8, of a section
        int has = -1;
        for (; gi < g1; gi += kAhead * kLoraWarps) {
#pragma unroll
            for (int d = 0; d < kAhead; ++d) {
                if (gi + d * kLoraWarps >= g1) break;
                if (ahead[d].section != has) {
                    has = ahead[d].section;
                    const T* h_row = hi_s + g * p.h_stride + has * p.R + 4 * j;
                    if (4 * j < p.R) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            h[half][0] = *reinterpret_cast<const uint2*>(h_row + half * lo_at);
                            h[half][1] = *reinterpret_cast<const uint2*>(h_row + half * lo_at + 8 * p.h_stride);
                        }
                    }
                }
                float acc[4][4];
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int t = 0; t < 4; ++t) mma_16816<T>(acc[t], h[half][0].x, h[half][1].x, h[half][0].y, h[half][1].y, next_s[d][t].x, next_s[d][t].y);
                put(ahead[d], next_y[d], acc);
                if (gi + (d + kAhead) * kLoraWarps < g1) {
                    ahead[d] = group(gi + (d + kAhead) * kLoraWarps);
                    ask_s(ahead[d], next_s[d]);
                    ask_y(ahead[d], next_y[d]);
                }
            }
        }
        lora_cluster_wait();  // no CTA leaves while another may read its sums
        return;
    }
    for (; gi < g1; gi += kLoraWarps) {
        const Group now = ahead[0];
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
                yv[0] = next_y[0][0];
                yv[1] = next_y[0][1];
            }
            if (k0 + 32 * kChunks < p.R) {
                ask_w(now, k0 + 32 * kChunks);
            } else if (gi + kLoraWarps < g1) {
                ahead[0] = group(gi + kLoraWarps);
                ask_w(ahead[0], 0);
                ask_y(ahead[0], next_y[0]);
            }
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int k = k0 + 32 * c;
                if (k >= p.R) break;
                const bool in = k + 8 * j < p.R;  // R is a multiple of 8
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint4 top = make_uint4(0, 0, 0, 0), bottom = make_uint4(0, 0, 0, 0);
                    if (in) top = *reinterpret_cast<const uint4*>(h_row + k + half * lo_at);
                    if (in) bottom = *reinterpret_cast<const uint4*>(h_row + k + half * lo_at + 8 * p.h_stride);
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        mma_16816<T>(acc[t], top.x, bottom.x, top.y, bottom.y, wv[t][c].x, wv[t][c].y);
                        mma_16816<T>(acc[t], top.z, bottom.z, top.w, bottom.w, wv[t][c].z, wv[t][c].w);
                    }
                }
            }
        }
        put(now, yv, acc);
    }
    lora_cluster_wait();  // no CTA leaves while another may read its sums
}

// ------------------------------------------------------------------------------------------------ more rows: blocks of 128, h through memory
// A block's note: its first row where its rows are neighbours, or a few rows or many that lie apart.
constexpr int kLoraFew = -1, kLoraApart = -2;

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
    const int ranks = p.S * p.R, n_mma = (ranks + 15) & ~15, section_ranks = (p.R + 15) & ~15, pad = section_ranks - p.R;
    const uint32_t cta = lora_cluster_rank(), ctas = lora_cluster_size();
    const int unit = blockIdx.x / ctas;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (unit >= *p.n_blocks) return;
    const GroupBlock blk = p.blocks[unit];
    if (cta == 0 && tid == 0) {  // the rows of a block ascend
        const int first = p.rows[blk.first], last = p.rows[blk.first + blk.count - 1];
        p.blocks[unit].note = last - first == blk.count - 1 ? first : blk.count <= 32 ? kLoraFew : kLoraApart;
    }
    if (blk.key < 0) return;
    uint32_t cols = 32;
    while (cols < static_cast<uint32_t>(n_mma)) cols *= 2;
    if (tid == 0) {
        for (int i = 0; i < kLoraStages; ++i) tc::mbar_init(tc::smem_u32(bars + i), 1);
        tc::mbar_fence_init();
    }
    if (warp == 0) tc::tmem_alloc(tc::smem_u32(&tmem_slot), cols);
    if (tid < kLoraRows) rows_s[tid] = tid < blk.count ? p.rows[blk.first + tid] : -1;  // rows behind the last one: nobody reads their sums
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
    for (int i = 0; i < 4; ++i) xr[i] = rows_s[r0 + 32 * i] >= 0 ? static_cast<const T*>(p.x) + static_cast<size_t>(rows_s[r0 + 32 * i]) * p.K : nullptr;
    const int stages = p.stages;
    auto ask = [&](int step, int stage) {
        const uint32_t to = base + stage * stage_bytes;
        const int k = 64 * (s0 + step) + 8 * c;
        const bool in = k < p.K;
        const int from = in ? k : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (xr[i]) lora_copy(to + lora_sw(r0 + 32 * i, c), xr[i] + from, in);
        for (int r = r0; r < ranks; r += 32) lora_copy(to + kLoraSub + lora_sw(r, c), a + static_cast<size_t>(r) * p.K + from, in);
    };
    for (int i = 0; i < stages - 1; ++i) {
        if (i < steps) ask(i, i);
        lora_commit();
    }
    bool broken = false;
    const uint32_t idesc = tc::instr_desc(lora_fmt<T>(), lora_fmt<T>(), 128, static_cast<uint32_t>(n_mma));
    int stage = 0, before = 0;      // of this step, of the step before
    uint32_t phase = 0, phase_before = 0;
    for (int step = 0; step < steps; ++step) {
        // (the group of this step is the one behind stages - 2 younger ones)
        if (stages == 3) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group %0;" ::"n"(kLoraStages - 2) : "memory");
        lora_proxy_fence();
        __syncthreads();
        if (tid == 0) {
            const uint32_t at = base + stage * stage_bytes;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
                tc::mma_f16(tmem, tc::smem_desc_k_sw128(at + ks * 32), tc::smem_desc_k_sw128(at + kLoraSub + ks * 32), idesc, step > 0 || ks > 0);
            tc::mma_commit(bar0 + 8 * stage);
        }
        // the stage that the step before this one read is filled again
        if (step > 0 && !lora_mma_done(bar0 + 8 * before, phase_before, broken, p.status)) broken = true;
        if (step + stages - 1 < steps) ask(step + stages - 1, step > 0 ? before : stages - 1);
        lora_commit();
        before = stage;
        phase_before = phase;
        if (++stage == stages) {
            stage = 0;
            phase ^= 1;
        }
    }
    if (steps > 0 && !lora_mma_done(bar0 + 8 * before, phase_before, broken, p.status)) broken = true;
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
        T* hi = static_cast<T*>(p.hi) + static_cast<size_t>(blk.first + r) * p.S * section_ranks;
        T* lo = static_cast<T*>(p.lo) + static_cast<size_t>(blk.first + r) * p.S * section_ranks;
        const float mul = lora_join<T, kLoraWideRanks>(part + r * pitch, ranks, ctas, scaling, [&](int n, T vh, T vl) {
            const int to = n + n / p.R * pad;
            hi[to] = vh;
            lo[to] = vl;
        });
        if (pad)  // eight ranks behind each section's: zeros, the MMA takes sixteen at a time
            for (int i = lane; i < 8 * p.S; i += 32) {
                const int to = (i >> 3) * section_ranks + p.R + (i & 7);
                hi[to] = lo[to] = from_float<T>(0.f);
            }
        if (lane == 0) p.mul[blk.first + r] = mul;
    }
    lora_cluster_arrive();
    lora_cluster_wait();
}

// ---- y + B h in tiles of 128 rows x 128 columns
constexpr int kLoraExpandThreads = 320;
constexpr int kLoraTileY = 2 * kLoraSub;             // a y tile: two halves of 64 columns, swizzled
constexpr int kLoraMostY = 4, kLoraMostB = 3;

// Rings of y tiles, of B tiles (`steps` x 64 ranks), and h (value and remainder), in shared memory.
struct LoraExpandLayout {
    int ys, bs, b_bytes, h_bytes;
    size_t smem;
};
__host__ __device__ inline LoraExpandLayout lora_layout(int steps) {
    LoraExpandLayout v;
    v.ys = steps == 1 ? 4 : 3;
    v.bs = steps == 1 ? 3 : 1;
    v.b_bytes = steps * kLoraSub;
    v.h_bytes = 2 * steps * kLoraSub;
    v.smem = 1024 + static_cast<size_t>(v.ys) * kLoraTileY + static_cast<size_t>(v.bs) * v.b_bytes + v.h_bytes;
    return v;
}

__device__ __forceinline__ void lora_tma_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar),
                 "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
__device__ __forceinline__ void lora_bulk_in(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void lora_tma_store(const CUtensorMap* map, int c0, int c1, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(c0), "r"(c1) : "memory");
}

// The n-th use of a ring of `size` barriers.
__device__ __forceinline__ bool lora_ring_wait(uint32_t ring, int n, int size) { return tc::mbar_wait(ring + 8 * (n % size), static_cast<uint32_t>((n / size) & 1)); }

// What the copying warp tells the others about a tile.
struct LoraTile {
    int32_t live;                    // 0: no more tiles
    int32_t mma;                     // which of the CTA's products the tile's is; -1: none
    int32_t first, cols;             // columns
    int32_t count, note;             // the block's
    int32_t row[kLoraRows];
    float mul[kLoraRows];
};
struct LoraProduct {
    int32_t live, new_h, last_h;     // the first and the last one that reads h as it is
};

// A CTA takes runs of neighbouring tiles; the runs are dealt over the CTAs, so that blocks of few rows and of many mix.
// Warp 0 brings y, B and (when the run, the block or the section changes) h by TMA and notes what a tile is; warp 1 issues the MMAs, h as two operands
// against the same B, into one of two accumulators; warps 2 to 9 add the sums to y where it lies (a row a lane, two warps a row quarter) and send the
// parts out by TMA.  Everything but the additions is asynchronous, so one CTA an SM with two or three tiles on their way is bound by memory.  (A second
// eight of adding warps gained nothing.)
// That is for blocks whose rows are neighbours, a prompt's.  A few rows that lie apart, requests that decode, come by a bulk copy each
// (about 50 cycles a copy: for all rows the same prompt took 532 us); of more, and at ragged ends, a lane reads and writes its row's 128 bytes itself.
// Waits are bounded.
template <typename T>
__global__ void __launch_bounds__(kLoraExpandThreads, 1)
    lora_expand_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_hi, const __grid_constant__ CUtensorMap map_lo,
                       const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_out, const __grid_constant__ LoraParams p) {
    extern __shared__ __align__(128) unsigned char smem_raw[];
    __shared__ LoraTile notes[kLoraMostY];
    __shared__ LoraProduct products[kLoraMostB];
    __shared__ __align__(8) uint64_t bars[2 * kLoraMostY + 2 * kLoraMostB + 4 + 2];
    __shared__ uint32_t tmem_slot;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int steps = (p.R + 63) / 64, section_ranks = (p.R + 15) & ~15;
    const LoraExpandLayout lay = lora_layout(steps);
    const uint32_t y_at = (tc::smem_u32(smem_raw) + 1023) & ~1023u, b_at = y_at + lay.ys * kLoraTileY, h_at = b_at + lay.bs * lay.b_bytes;
    const uint32_t y_full = tc::smem_u32(bars), y_free = y_full + 8 * kLoraMostY, b_full = y_free + 8 * kLoraMostY, b_free = b_full + 8 * kLoraMostB;
    const uint32_t acc_full = b_free + 8 * kLoraMostB, acc_free = acc_full + 16, h_full = acc_free + 16, h_free = h_full + 8;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kLoraMostY; ++i) {
            tc::mbar_init(y_full + 8 * i, 1);
            tc::mbar_init(y_free + 8 * i, 8);
        }
        for (int i = 0; i < kLoraMostB; ++i) {
            tc::mbar_init(b_full + 8 * i, 1);
            tc::mbar_init(b_free + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(acc_full + 8 * i, 1);
            tc::mbar_init(acc_free + 8 * i, 8);
        }
        tc::mbar_init(h_full, 1);
        tc::mbar_init(h_free, 1);
        tc::mbar_fence_init();
    }
    if (warp == 1) tc::tmem_alloc(tc::smem_u32(&tmem_slot), 2 * kLoraTile);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    // with the TMEM columns in hand: a dependent grid that took them first and then waited for this one would never give them back
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) {
        // ---- copies in
        const int tiles = p.tile_ends[p.S - 1], n_blocks = *p.n_blocks;
        const int64_t step = static_cast<int64_t>(gridDim.x - 1) * p.run + 1;  // from the last tile of a run to the first of the next
        const int step_blocks = static_cast<int>(step / tiles), step_tiles = static_cast<int>(step % tiles);
        int block = static_cast<int>(static_cast<int64_t>(blockIdx.x) * p.run / tiles), t = static_cast<int>(static_cast<int64_t>(blockIdx.x) * p.run % tiles);
        int left = p.run, section = 0, n = 0, n_b = 0, n_h = 0;  // left: tiles of the run, this one included
        bool new_block = true, new_h = true;                     // since the tile before
        GroupBlock blk = {};
        int row[4] = {};
        float mul[4] = {};
        bool ok = true;
        for (; block < n_blocks; ++n) {
            while (t >= p.tile_ends[section]) ++section;
            const int first = (section ? p.ends[section - 1] : 0) + kLoraTile * (t - (section ? p.tile_ends[section - 1] : 0));
            const int cols = min(kLoraTile, p.ends[section] - first), halves = cols > 64 ? 2 : 1;
            if (new_block) {
                blk = p.blocks[block];
                // neighbouring rows need no list, and a factor is one in bf16
                if (blk.note < 0 || std::is_same<T, __half>::value) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int r = lane + 32 * q;
                        row[q] = r < blk.count ? p.rows[blk.first + r] : 0;
                        mul[q] = r < blk.count && blk.key >= 0 ? p.mul[blk.first + r] : 0.f;
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        row[q] = blk.note + lane + 32 * q;
                        mul[q] = 1.f;
                    }
                }
            }
            const bool adds = blk.key >= 0;
            // h is asked for anew with every run, block and section, and given back with the last tile before the next: what that is, is known here
            const bool last_h = left == 1 || t + 1 == p.tile_ends[section];
            const int sb = n_b % lay.bs, sy = n % lay.ys;
            if (adds && n_b >= lay.bs) ok = lora_ring_wait(b_free, n_b - lay.bs, lay.bs);
            if (ok && adds && new_h && n_h > 0) ok = lora_ring_wait(h_free, n_h - 1, 1);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            if (adds) {
                if (lane == 0) {
                    products[sb].live = 1;
                    products[sb].new_h = new_h;
                    products[sb].last_h = last_h;
                    tc::mbar_expect_tx(b_full + 8 * sb, lay.b_bytes);
                    for (int k = 0; k < steps; ++k) lora_tma_3d(b_at + sb * lay.b_bytes + k * kLoraSub, &map_b, 64 * k, first, blk.key, b_full + 8 * sb);
                    if (new_h) {
                        tc::mbar_expect_tx(h_full, lay.h_bytes);
                        for (int k = 0; k < steps; ++k) {
                            tc::tma_load_2d(h_at + 2 * k * kLoraSub, &map_hi, section * section_ranks + 64 * k, blk.first, h_full);
                            tc::tma_load_2d(h_at + (2 * k + 1) * kLoraSub, &map_lo, section * section_ranks + 64 * k, blk.first, h_full);
                        }
                    }
                }
                ++n_b;
                n_h += new_h;
            }
            if (n >= lay.ys) ok = lora_ring_wait(y_free, n - lay.ys, lay.ys);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            LoraTile& note = notes[sy];
            if (lane == 0) {
                note.live = 1;
                note.mma = adds ? n_b - 1 : -1;
                note.first = first;
                note.cols = cols;
                note.count = blk.count;
                note.note = blk.note;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                note.row[lane + 32 * q] = row[q];
                note.mul[lane + 32 * q] = mul[q];
            }
            __syncwarp();
            const uint32_t bar = y_full + 8 * sy, to = y_at + sy * kLoraTileY;
            if (lane == 0) {
                tc::mbar_expect_tx(bar, blk.note >= 0 ? halves * kLoraSub : blk.note == kLoraFew ? blk.count * cols * 2 : 0);
                if (blk.note >= 0)
                    for (int h = 0; h < halves; ++h) tc::tma_load_2d(to + h * kLoraSub, &map_y, first + 64 * h, blk.note, bar);
            }
            if (blk.note == kLoraFew) {
                __syncwarp();  // behind the bytes that are expected
                if (lane < blk.count)
                    for (int h = 0; h < halves; ++h)
                        lora_bulk_in(to + h * kLoraSub + lane * 128, static_cast<const T*>(p.y) + static_cast<size_t>(row[0]) * p.N + first + 64 * h, 2 * min(64, cols - 64 * h), bar);
            }
            // the next tile
            new_block = false;
            new_h = last_h;
            if (--left == 0) {
                left = p.run;
                block += step_blocks;
                t += step_tiles;
                section = 0;
                new_block = step_blocks > 0;
            } else {
                ++t;
            }
            if (t >= tiles) {
                t -= tiles;
                ++block;
                section = 0;
                new_block = true;
            }
        }
        // the end
        if (ok && n_b >= lay.bs) ok = lora_ring_wait(b_free, n_b - lay.bs, lay.bs);
        if (ok && lane == 0) {
            products[n_b % lay.bs].live = 0;
            tc::mbar_arrive(b_full + 8 * (n_b % lay.bs));
        }
        if (ok && n >= lay.ys) ok = lora_ring_wait(y_free, n - lay.ys, lay.ys);
        if (ok && lane == 0) {
            notes[n % lay.ys].live = 0;
            tc::mbar_arrive(y_full + 8 * (n % lay.ys));
        }
        if (!ok && lane == 0) {  // nothing may land behind the CTA's end
            atomicExch(p.status, 1);
            for (int i = n < lay.ys ? 0 : n - lay.ys; i < n; ++i) lora_ring_wait(y_full, i, lay.ys);
            for (int i = n_b < lay.bs ? 0 : n_b - lay.bs; i < n_b; ++i) lora_ring_wait(b_full, i, lay.bs);
            if (n_h > 0) lora_ring_wait(h_full, n_h - 1, 1);
        }
    } else if (warp == 1) {
        // ---- MMAs
        if (lane == 0) {
            const uint32_t idesc = tc::instr_desc(lora_fmt<T>(), lora_fmt<T>(), 128, kLoraTile);
            int n_h = 0, n = 0;
            for (;; ++n) {
                const int s = n % lay.bs;
                bool ok = lora_ring_wait(b_full, n, lay.bs);
                if (ok && !products[s].live) break;
                const bool last_h = ok && products[s].last_h;
                if (ok && products[s].new_h) ok = lora_ring_wait(h_full, n_h++, 1);
                if (ok && n >= 2) ok = lora_ring_wait(acc_free, n - 2, 2);
                if (!ok) {
                    atomicExch(p.status, 2);
                    break;
                }
                tc::fence_after_sync();
                const uint32_t d = tmem + kLoraTile * (n & 1), w_at = b_at + s * lay.b_bytes;
                for (int k = 0; k < section_ranks / 16; ++k) {
                    const uint32_t a = h_at + (k >> 2) * 2 * kLoraSub + (k & 3) * 32;
                    const uint64_t w = tc::smem_desc_k_sw128(w_at + (k >> 2) * kLoraSub + (k & 3) * 32);
                    tc::mma_f16(d, tc::smem_desc_k_sw128(a), w, idesc, k > 0);
                    tc::mma_f16(d, tc::smem_desc_k_sw128(a + kLoraSub), w, idesc, true);
                }
                if (last_h) tc::mma_commit(h_free);
                tc::mma_commit(b_free + 8 * s);
                tc::mma_commit(acc_full + 8 * (n & 1));
            }
            if (n > 0) lora_ring_wait(acc_full, n - 1, 2);  // nothing in flight when the columns are given back
        }
    } else {
        // ---- sums, a row a lane
        const int quarter = warp & 3, half = (warp - 2) >> 2, r = 32 * quarter + lane;
        for (int n = 0;; ++n) {
            const int s = n % lay.ys;
            if (!__all_sync(0xFFFFFFFFu, lora_ring_wait(y_full, n, lay.ys))) {
                if (lane == 0) atomicExch(p.status, 3);
                break;
            }
            const LoraTile& note = notes[s];
            if (!note.live) break;
            const int mma = note.mma, count = note.count, where = note.note, first = note.first + 64 * half;
            const int bytes = min(128, 2 * note.cols - 128 * half);  // of this warp's columns
            const bool has = r < count, here = where != kLoraApart, whole = where >= 0 && bytes == 128 && 32 * quarter + 32 <= count;
            const bool mine = 32 * quarter < count && bytes > 0;  // of the whole warp
            const int turn = where >= 0 ? r & 7 : 0;  // TMA has swizzled the tile, bulk copies of rows have not
            const uint32_t part = y_at + s * kLoraTileY + half * kLoraSub, at = part + r * 128;
            const size_t to = static_cast<size_t>(note.row[r]) * p.N + first;
            const float mul = note.mul[r];
            uint4 y[8];
            if (mine) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    if (here)
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(y[c].x), "=r"(y[c].y), "=r"(y[c].z), "=r"(y[c].w) : "r"(at + ((c ^ turn) << 4)) : "memory");
                    else if (has && 16 * c < bytes)
                        y[c] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.y) + to + 8 * c);
                }
            }
            if (mma >= 0) {
                if (!lora_ring_wait(acc_full, mma, 2)) atomicExch(p.status, 3);
                __syncwarp();
                if (mine) {
                    tc::fence_after_sync();
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t v[32];
                        tc::tmem_ld_32x32(tmem + ((32u * quarter) << 16) + kLoraTile * (mma & 1) + 64 * half + 32 * h, v);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t* e = reinterpret_cast<uint32_t*>(&y[4 * h + c]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) e[i] = lora_add2<T>(e[i], __uint_as_float(v[8 * c + 2 * i]), __uint_as_float(v[8 * c + 2 * i + 1]), mul);
                        }
                    }
                }
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(acc_free + 8 * (mma & 1));
            }
            if (mine && whole) {
                if (mma >= 0) {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        asm volatile("st.shared.v4.u32 [%4], {%0,%1,%2,%3};" ::"r"(y[c].x), "r"(y[c].y), "r"(y[c].z), "r"(y[c].w), "r"(at + ((c ^ turn) << 4)) : "memory");
                    lora_proxy_fence();
                    __syncwarp();
                }
                if (lane == 0) {
                    lora_tma_store(&map_out, first, where + 32 * quarter, part + 32 * quarter * 128);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            } else if (mine && has) {
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (16 * c < bytes) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + to + 8 * c) = y[c];
            }
            // the slot is free once its rows have been read, by the lanes and by the copy out
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(y_free + 8 * s);
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 1) tc::tmem_dealloc(tmem, 2 * kLoraTile);
}

static size_t lora_align(size_t v) { return (v + 255) / 256 * 256; }

static bool lora_wide(int64_t S, int64_t R) { return R <= kLoraWideRank && S <= kLoraMaxSections && S * R <= kLoraWideRanks; }

// Rows of a block.  Above kLoraSelfPlan rows, 16 (lora_rows_kernel reads a block's A and B from L2 again for every 16 rows, and has one launch behind the list) up to
// T (K + 2 N) max(R, 32) = 2 10^9 for sixteen ranks in all, 8 10^8 for more; 128 from there on.  The line is where prompts cross.  Requests that decode fill few rows of a
// block of 128, and with many adapters blocks of 16 would be faster far beyond it; but how the rows lie is not known on the host.  Both forced, 16 : 128, us, prompts of 3
// adapters | 100 rows that decode, of 16 adapters, and prompts | rows that decode in any order, of 16 | of 64; in brackets the expression in 10^9:
//   K=N=4096, rank 16         600 rows (0.2) 11 : 23 | 11 : 33 | 12 : 31 | 17 : 61, 2400 (0.9) 35 : 34 | 34 : 42 | 33 : 59 | 36 : 88, 4800 (1.9) 54 : 50 | 53 : 50 | 53 : 83 | 56 : 87,
//                             6000 (2.4) 59 : 54 | 59 : 58 | 61 : 88 | 64 : 94
//   K=4096 N=28672, rank 16   300 rows (0.6) 20 : 31 | 21 : 72 | 25 : 84 | 42 : 186, 900 (1.8) 35 : 44 | 39 : 84 | 48 : 85 | 73 : 244, 1200 (2.4) 56 : 49 | 60 : 89 | 74 : 95 | 77 : 275,
//                             2400 (4.7) 105 : 71 | 109 : 114 | 121 : 177 | 126 : 300
//   K=14336 N=4096, rank 16   1200 rows (0.9) 27 : 37 | 28 : 46 | 27 : 49 | 30 : 117, 2400 (1.7) 52 : 45 | 52 : 64 | 39 : 70 | 55 : 128, 3600 (2.6) 59 : 53 | 59 : 69 | 60 : 85 | 63 : 121
//   K=N=4096, rank 32         1200 rows (0.5) 22 : 27 | 22 : 35 | 23 : 38 | 25 : 78, 1800 (0.7) 23 : 29 | 24 : 37 | 25 : 42 | 27 : 87, 2400 (0.9) 43 : 34 | 43 : 38 | 35 : 60 | 46 : 89
//   K=N=4096, rank 64         600 rows (0.5) 21 : 23 | 22 : 35 | 22 : 33 | 34 : 65, 900 (0.7) 22 : 25 | 24 : 38 | 24 : 36 | 35 : 74, 1200 (0.9) 34 : 27 | 35 : 37 | 33 : 40 | 38 : 81
//   K=4096 N=28672, rank 64   300 rows (1.2) 40 : 33 | 40 : 75 | 41 : 85 | 68 : 193, 600 (2.4) 68 : 38 | 69 : 77 | 70 : 90 | 118 : 219
//   K=N=5120, rank 128        300 rows (0.6) 26 : 26 | 27 : 41 | 27 : 43 | 41 : 84, 1200 (2.4) 66 : 34 | 67 : 45 | 62 : 55 | 72 : 107
static int lora_block_rows(int64_t T, int64_t K, int64_t N, int64_t S, int64_t R) {
    if (T <= kLoraSelfPlan || !lora_wide(S, R)) return 16;
    return static_cast<double>(T) * (K + 2 * N) * (R < 32 ? 32 : R) < (S * R <= 16 ? 2e9 : 8e8) ? 16 : kLoraRows;
}
static bool lora_self(int64_t T, int block_rows) { return block_rows == 16 && T <= kLoraSelfRows; }
static int64_t lora_units(int64_t T, int64_t L, int block_rows) { return group_max_blocks(T, L, block_rows, block_rows == kLoraRows); }

// CTAs of a cluster: the largest of 8, 4, 2, 1 with which so many blocks stay within `most` CTAs an SM, and two within `pairs`.
static int lora_cluster(int64_t blocks, int64_t most, int64_t pairs) {
    int ctas = 8;
    while (ctas > 1 && blocks * ctas > (ctas > 2 ? most : pairs) * sm_count()) ctas /= 2;
    return ctas;
}
// Blocks of 16 rows that a call is likely to have: the kinds of rows that T draws out of L + 1 meet, with one block each or half a block more than they fill.
static int64_t lora_likely_blocks(int64_t T, int64_t L) {
    const double kinds = static_cast<double>(L + 1), met = kinds * (1 - exp(-T / kinds)), filled = T / met / 16 + 0.5;
    return static_cast<int64_t>(ceil(met * (filled < 1 ? 1 : filled)));
}
// Within two CTAs an SM, which run at once; projections of 5120 columns and more keep two a block up to four an SM.  us with clusters of 1, 2, 4, 8, the one that is
// taken in brackets:
//   K=N=4096, rank 16             64 rows of 64 adapters 15.7 11.3 [8.5] 12.3, 256 of 8 16.7 11.3 8.5 [7.9], 256 of 64 18.4 12.3 [9.9] 15.7, 256 of 400 [23.6] 26.3 26.6 41.3
//     prompts of three            500 rows 17.1 12.6 9.9 [10.2], 700 19.5 13.7 [10.9] 16.0, 1200 23.9 [17.7] 20.5 25.3, 2000 26.3 [19.8] 24.9 39.9, 3200 [33.1] 37.9 37.5 56.0
//   K=14336 N=4096, rank 16       64 of 64 31.1 19.1 [13.0] 16.7, 200 of 200 37.9 [24.2] 27.6 37.9, 256 of 400 [39.9] 43.0 40.3 54.3
//   K=4096 N=28672, rank 64       64 of 64 163 103 [64] 68, 128 of 128 196 [116] 112 100, 256 of 64 178 108 [71] 78, 256 of 400 225 [209] 179 193
// and 1 : 2 with more blocks than SMs, 256 rows of 256 and of 400 adapters, 2400 mixed rows of 100, rank 16: K=1024 N=1024 9 : 11, 9 : 13, 16 : 19, N=4096 17 : 17, 18 : 21, 28 : 30,
// N=5120 26 : 22, 28 : 23, 33 : 37, N=8192 37 : 27, 38 : 30, 43 : 44; K=4096 N=4096 23 : 23, 24 : 26, 32 : 35, N=8192 38 : 31, 39 : 36, 47 : 48.
static int lora_rows_cluster(int64_t T, int64_t L, int64_t N) { return lora_cluster(lora_likely_blocks(T, L), 2, N >= 5120 ? 4 : 2); }

static int lora_launch(void (*kernel)(const LoraParams), const LoraParams& p, int64_t grid, int cluster, size_t smem, cudaStream_t stream) {
    if (smem > kSmemUnasked) EQ_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024));
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
    const int ranks = p.S * p.R, section_ranks = (p.R + 15) & ~15;
    const int block_rows = lora_block_rows(p.T, p.K, p.N, p.S, p.R);
    const int64_t units = lora_units(T_, L, block_rows);
    const bool self = lora_self(p.T, block_rows);
    p.status = p.T > kLoraSelfPlan ? reinterpret_cast<int*>(base) : nullptr;
    if (!self) {
        size_t o = 256;
        auto take = [&](size_t bytes) {
            void* at = base + o;
            o += lora_align(bytes);
            return at;
        };
        int32_t* n_blocks = reinterpret_cast<int32_t*>(base) + 1;
        GroupBlock* blocks = static_cast<GroupBlock*>(take(static_cast<size_t>(units) * sizeof(GroupBlock)));
        int32_t* rows = static_cast<int32_t*>(take(static_cast<size_t>(T_) * 4));
        p.blocks = blocks;
        p.n_blocks = n_blocks;
        p.rows = rows;
        const int st = group_rows_launch(p.ids, p.T, p.L, !p.in_place, block_rows, block_rows == kLoraRows, blocks, n_blocks, rows, p.status, stream);
        if (st != EQ_OK) return st;
        if (block_rows == kLoraRows) {
            p.mul = static_cast<float*>(take(static_cast<size_t>(T_) * 4));
            p.hi = take(static_cast<size_t>(T_) * p.S * section_ranks * 2);
            p.lo = take(static_cast<size_t>(T_) * p.S * section_ranks * 2);
        }
    }
    if (block_rows == 16) {
        p.h_stride = (ranks + 63) / 64 * 64 + 32;  // rows 64 bytes apart modulo 128: the 16-byte reads of two rows meet every bank once
        const size_t red = static_cast<size_t>(kLoraWarps) * 16 * (kLoraPass + 8) * sizeof(float), split = 2 * static_cast<size_t>(16) * p.h_stride * 2;
        const int ctas = lora_rows_cluster(T_, L, p.N);
        const size_t counts = p.blocks || p.T <= 32 ? 0 : (static_cast<size_t>(L) + 1) * (p.T > kLoraSelfPlan ? sizeof(uint4) : sizeof(uint2));
        const size_t work = static_cast<size_t>(16) * ranks * sizeof(float) + (red > split ? red : split);
        return lora_launch(ranks <= 16 ? lora_rows_kernel<T, 1, true> : p.R <= 32 ? lora_rows_kernel<T, 1, false> : lora_rows_kernel<T, 2, false>, p, units * ctas, ctas,
                           work > counts ? work : counts, stream);
    }
    // Steps ahead: six where two CTAs an SM have room for them.  24 adapters of rank 16, prompts, us a call with three and with six: 8192 rows of K=N=5120
    // 82 and 73, 4096 of K=14336 N=5120 75 and 64.
    p.stages = kLoraStages * (kLoraSub + lora_stage_rows(ranks)) <= 110 * 1024 ? kLoraStages : 3;
    const size_t stages = p.stages * (kLoraSub + lora_stage_rows(ranks)), sums = static_cast<size_t>(kLoraRows) * (ranks + 4) * sizeof(float);
    // (a shrink of blocks of 128 rows, three CTAs an SM: with at most 1, 2, 3, 4, 8, us a call, 8192 rows of two adapters, K=4096 N=28672, rank 64, 220 208 208 216 216; of
    // 24, rank 16, 4096 rows of K=14336 N=5120 156 95 65 65 62, 8192 of K=N=5120 108 87 87 90 89)
    const int ctas = lora_cluster(units, 3, 3);
    const int st = lora_launch(lora_shrink_kernel<T>, p, units * ctas, ctas, 1024 + (stages > sums ? stages : sums), stream);
    if (st != EQ_OK) return st;
    const CUtensorMapDataType elem = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUtensorMap map_b, map_hi, map_lo, map_y, map_out;
    int mt = make_tensor_map_3d(&map_b, p.b, elem, 2, p.L, p.N, p.R, kLoraTile, 64, CU_TENSOR_MAP_SWIZZLE_128B);
    const uint64_t h_cols = static_cast<uint64_t>(p.S) * section_ranks;
    if (mt == EQ_OK) mt = make_tensor_map_2d(&map_hi, p.hi, elem, 2, p.T, h_cols, h_cols * 2, kLoraRows, 64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (mt == EQ_OK) mt = make_tensor_map_2d(&map_lo, p.lo, elem, 2, p.T, h_cols, h_cols * 2, kLoraRows, 64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (mt == EQ_OK) mt = make_tensor_map_2d(&map_y, p.y, elem, 2, p.T, p.N, static_cast<uint64_t>(p.N) * 2, kLoraRows, 64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (mt == EQ_OK) mt = make_tensor_map_2d(&map_out, p.out, elem, 2, p.T, p.N, static_cast<uint64_t>(p.N) * 2, 32, 64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (mt != EQ_OK) return mt;
    const LoraExpandLayout lay = lora_layout((p.R + 63) / 64);
    // a CTA's tiles: runs of four where that leaves at least two runs a CTA, fewer where there are few tiles
    const int64_t all_tiles = units * p.tile_ends[p.S - 1];
    p.run = static_cast<int>(all_tiles / (2 * sm_count()) < 1 ? 1 : all_tiles / (2 * sm_count()) > 4 ? 4 : all_tiles / (2 * sm_count()));
    const int64_t runs = ceil_div(all_tiles, p.run);
    EQ_CUDA_OK(cudaFuncSetAttribute(lora_expand_kernel<T>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    EQ_CUDA_OK(cudaFuncSetAttribute(lora_expand_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lay.smem)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(runs < sm_count() ? runs : sm_count()));
    cfg.blockDim = dim3(kLoraExpandThreads);
    cfg.dynamicSmemBytes = lay.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    EQ_CUDA_OK(cudaLaunchKernelEx(&cfg, lora_expand_kernel<T>, map_b, map_hi, map_lo, map_y, map_out, static_cast<const LoraParams&>(p)));
    return EQ_OK;
}

}  // namespace eq

using namespace eq;

extern "C" size_t eq_lora_workspace_bytes(int64_t T, int64_t L, int64_t S, int64_t R) {
    if (T <= kLoraSelfPlan || L <= 0 || S <= 0 || R <= 0) return 0;
    const int64_t few = lora_units(T, L, 16), many = lora_units(T, L, kLoraRows);
    const size_t lists = 256 + lora_align(static_cast<size_t>(few > many ? few : many) * sizeof(GroupBlock)) + lora_align(static_cast<size_t>(T) * 4);
    return !lora_wide(S, R) ? lists : lists + lora_align(static_cast<size_t>(T) * 4) + 2 * lora_align(static_cast<size_t>(T) * S * ((R + 15) / 16 * 16) * 2);
}

extern "C" const char* eq_lora_kernel(int64_t T, int64_t K, int64_t N, int64_t R, int64_t S) {
    const int block_rows = lora_block_rows(T, K, N, S, R);
    return block_rows == kLoraRows ? "lora_expand_kernel" : lora_self(T, block_rows) ? "lora_rows_kernel" : "group_rows_kernel + lora_rows_kernel";
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
    // CTAs write rows of out while others read x, A, B and their rows of y
    const uintptr_t out0 = reinterpret_cast<uintptr_t>(out), out1 = out0 + static_cast<size_t>(T) * N * 2;
    auto apart = [&](const void* from, size_t bytes) { return reinterpret_cast<uintptr_t>(from) >= out1 || reinterpret_cast<uintptr_t>(from) + bytes <= out0; };
    EQ_REQUIRE((out == y || apart(y, static_cast<size_t>(T) * N * 2)) && apart(x, static_cast<size_t>(T) * K * 2) && apart(a, static_cast<size_t>(L) * S * R * K * 2) &&
                   apart(b, static_cast<size_t>(L) * N * R * 2) && apart(scaling, static_cast<size_t>(L) * 4) && apart(adapter_ids, static_cast<size_t>(T) * 4) &&
                   (need == 0 || apart(workspace, need)),
               EQ_ERR_BAD_ARG, "eq_lora_add: out may be y and overlaps no other argument");
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
