// Routed MoE layer of a few tokens on FP8 (e4m3) experts, weights as the checkpoint stores them:
//     y[t] = sum_j p[t, j] W_down[e] (silu(W_gate[e] x[t]) * (W_up[e] x[t])),  e = id[t, j],
// id the topk experts of largest router logit (ties to the lowest id), p their softmax, renormalised over the picks.
// Activations keep their 16 bits (a decode batch is bound by the weights' bytes: quantizing them would cost accuracy and buy nothing);
// a weight is bits x scale, the scale per output channel or per 128 x 128 block, applied to f32 sums.  The products of a 128-element block of K are
// summed by mma.sync in f32, the blocks added in f32.  silu(gate) * up is kept as two 16-bit numbers (value and remainder), so that the
// layer rounds once, as y is stored.
//
// Up to 32 tokens and 256 experts, two launches:
//   gate_up  Every CTA routes the tokens and groups the picks by expert itself: a block is at most eight rows (picks) of one expert, so
//            an expert that several tokens picked is read once.  The blocks' tiles of eight gate and the same eight up rows (one MMA
//            A operand of sixteen rows, the block's rows as the N = 8 columns) are one stream, cut into equal spans over the CTAs and
//            in a CTA into equal shares of 128-element items over its warps.  A tile's silu and product happen in the registers of whoever
//            has its sums; tiles that several warps share meet in shared memory in warp order.
//   down     The second launch has routed the tokens and asked for its first weights before the first one ends.  A CTA has sixteen
//            output channels of ALL the blocks: the picks of a token meet inside it (f32, a fixed order), y is written once, and nothing is
//            combined across CTAs: no atomics, no counters, no rows in memory.
// Above, route + group.cu list the blocks, and both products run as streams of tiles; the down rows go to memory in f32 and
// moe_w8_combine_kernel adds them.
//
// Weights reach a lane through a ring in shared memory that the lane fills by cp.async for itself (16 bytes of a row: K indices 16 j .. 16 j + 15
// of each half of the item, in both operands alike), so no warp waits for another.  mma.sync and not tcgen05: with at most eight rows the weights'
// bytes bound the layer; an item of 2 KB is 8 MMAs (17 cycles of an SM's 2.1 each) beside the 89 cycles that HBM needs for it.
#include "group.cuh"
#include "mma_sync.cuh"

namespace eq {

constexpr int kW8Threads = 256;
constexpr int kW8Warps = kW8Threads / 32;
constexpr int kW8Depth = 5;             // items of a warp's ring
constexpr int kW8Item = 2048;           // sixteen rows x 128 elements
constexpr int kW8SelfTokens = 32;       // tokens up to which the CTAs route and group themselves (one bit each of a word)
constexpr int kW8SelfExperts = 256;
constexpr int kW8MaxTopK = 16;
constexpr int kW8SelfPicks = kW8SelfTokens * kW8MaxTopK;
constexpr int kW8BlockRows = 8;

struct W8Params {
    const uint8_t* w;         // this phase's weights: gate_up [E][2I][H] or down [E][H][I]
    const float* scale;       // [E][2I] / [E][H], or [E][2I / 128][H / 128] / [E][H / 128][I / 128]
    const float* logits;      // [T][E]
    const void* x;            // [T][H]
    void* hi;                 // [picks][I] silu(gate) * up, value
    void* lo;                 //            and remainder
    void* y;                  // [T][H]
    float* rows_out;          // [picks][H], general form
    const GroupBlock* blocks; // general form
    const int32_t* n_blocks;
    const int32_t* rows;      // pick of each row in expert order
    int T, E, topk, H, I;
};

// The picks in expert order, worked out by a CTA for itself.
struct W8Plan {
    uint32_t tokens[kW8SelfExperts];      // tokens that picked an expert
    uint16_t first_block[kW8SelfExperts];
    uint16_t first_row[kW8SelfExperts];
    int16_t id[kW8SelfPicks];             // [token][topk], -1: dropped
    float share[kW8SelfPicks];
    uint16_t expert[kW8SelfPicks];        // of a block
    uint16_t row0[kW8SelfPicks];
    uint8_t count[kW8SelfPicks];
    uint8_t token[kW8SelfPicks];          // of a row
    float score[kW8SelfPicks];
    int sums[2 * kW8Warps];
    int n_blocks;
};

// f32 -> a key whose unsigned order is the float order, equal for both zeros; 0 for a NaN, which is never picked.
__device__ __forceinline__ uint32_t w8_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v != v ? 0u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One warp, one token: picks in the order of their logits, and their shares.
__device__ __forceinline__ void w8_route(const float* __restrict__ logits, int E, int topk, int16_t* id, float* share) {
    constexpr int kNV = kW8SelfExperts / 32;
    const int lane = threadIdx.x & 31;
    uint32_t key[kNV];
    bool nan = false;
#pragma unroll
    for (int b = 0; b < kNV; ++b) {
        const float v = lane + 32 * b < E ? logits[lane + 32 * b] : 0.f;
        nan = nan || v != v;
        key[b] = lane + 32 * b < E ? w8_key(v) : 0u;
    }
    nan = __any_sync(0xFFFFFFFFu, nan);
    int my_id = -1;
    float my_v = 0.f, top = 0.f;
    for (int k = 0; k < topk; ++k) {
        uint32_t best = 0;
        int at = 0;
#pragma unroll
        for (int b = 0; b < kNV; ++b)
            if (key[b] > best) {
                best = key[b];
                at = b;
            }
        const uint32_t win = __reduce_max_sync(0xFFFFFFFFu, best);
        const uint32_t e = __reduce_min_sync(0xFFFFFFFFu, best == win && win ? static_cast<uint32_t>(lane + 32 * at) : 0xFFFFFFFFu);
        if (win && e == static_cast<uint32_t>(lane + 32 * at)) {
#pragma unroll
            for (int b = 0; b < kNV; ++b)
                if (b == at) key[b] = 0u;
        }
        const float value = __uint_as_float((win & 0x80000000u) ? (win & 0x7FFFFFFFu) : ~win);
        if (k == 0) top = value;
        if (win && lane == k) {
            my_id = static_cast<int>(e);
            my_v = value;
        }
    }
    float p = my_id >= 0 ? expf(my_v - top) : 0.f, sum = p;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
    if (lane == 0 && my_id < 0) my_id = E - 1;  // nothing but NaN: one pick, for the share below
    if (lane < topk) {
        id[lane] = static_cast<int16_t>(my_id);
        share[lane] = nan ? __int_as_float(0x7FC00000) : p / sum;  // the softmax of a row that holds a NaN
    }
}

__device__ __forceinline__ void w8_plan(const W8Params& p, W8Plan& plan) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    static_assert(kW8SelfExperts == kW8Threads, "an expert a thread");
    plan.tokens[tid] = 0;
    for (int t = warp; t < p.T; t += kW8Warps) w8_route(p.logits + static_cast<size_t>(t) * p.E, p.E, p.topk, plan.id + t * p.topk, plan.share + t * p.topk);
    __syncthreads();
    const int picks = p.T * p.topk;
    for (int i = tid; i < picks; i += kW8Threads)
        if (plan.id[i] >= 0) atomicOr(plan.tokens + plan.id[i], 1u << (i / p.topk));
    __syncthreads();
    const int c = __popc(plan.tokens[tid]), b = (c + kW8BlockRows - 1) / kW8BlockRows;
    int ci = c, bi = b;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int cu = __shfl_up_sync(0xFFFFFFFFu, ci, d), bu = __shfl_up_sync(0xFFFFFFFFu, bi, d);
        if (lane >= d) {
            ci += cu;
            bi += bu;
        }
    }
    if (lane == 31) {
        plan.sums[warp] = ci;
        plan.sums[kW8Warps + warp] = bi;
    }
    __syncthreads();
    int row = ci - c, block = bi - b;
    for (int w = 0; w < warp; ++w) {
        row += plan.sums[w];
        block += plan.sums[kW8Warps + w];
    }
    plan.first_row[tid] = static_cast<uint16_t>(row);
    plan.first_block[tid] = static_cast<uint16_t>(block);
    for (int r = 0; r < c; r += kW8BlockRows, ++block) {
        plan.expert[block] = static_cast<uint16_t>(tid);
        plan.row0[block] = static_cast<uint16_t>(row + r);
        plan.count[block] = static_cast<uint8_t>(min(kW8BlockRows, c - r));
    }
    if (tid == kW8Threads - 1) plan.n_blocks = block;
    __syncthreads();
    for (int i = tid; i < picks; i += kW8Threads) {
        const int e = plan.id[i], t = i / p.topk;
        if (e < 0) continue;
        const int at = plan.first_row[e] + __popc(plan.tokens[e] & ((1u << t) - 1));
        plan.token[at] = static_cast<uint8_t>(t);
        plan.score[at] = plan.share[i];
    }
    __syncthreads();
}

// Two e4m3 values (the low or the high half of a word) as a pair of the activations' type.
template <typename T>
__device__ __forceinline__ uint32_t w8_pair(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
    if (std::is_same<T, __half>::value) return h;
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    const __nv_bfloat162 r = __floats2bfloat162_rn(f.x, f.y);  // exact: e4m3 has four significant bits
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint4 w8_lds(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// One item: acc[16 rows][8 columns] += W x over 128 elements.  slot: this lane's first 16 bytes in the ring (top half of the item, rows g; then
// rows g + 8; then the bottom half's); b: the lane's column at the same K indices, sixteen values a half.
template <typename T, int SUBS>
__device__ __forceinline__ void w8_item(uint32_t slot, const uint4 (&b)[SUBS][4], float (&acc)[SUBS][4]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint4 top = w8_lds(slot + half * 1024), bottom = w8_lds(slot + half * 1024 + 512);
        const uint32_t t[4] = {top.x, top.y, top.z, top.w}, u[4] = {bottom.x, bottom.y, bottom.z, bottom.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t a0 = w8_pair<T>(t[q] & 0xFFFFu), a2 = w8_pair<T>(t[q] >> 16), a1 = w8_pair<T>(u[q] & 0xFFFFu), a3 = w8_pair<T>(u[q] >> 16);
#pragma unroll
            for (int s = 0; s < SUBS; ++s) {
                const uint4& v = b[s][2 * half + (q >> 1)];
                mma_16816<T>(acc[s], a0, a1, a2, a3, q & 1 ? v.z : v.x, q & 1 ? v.w : v.y);
            }
        }
    }
}

__device__ __forceinline__ void w8_copy(uint32_t to, const uint8_t* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void w8_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// A stream of items of a warp: tiles in order, each `items` items of 128 elements of K.  The owner says where a tile's rows lie for this lane.
struct W8Ring {
    uint32_t base, slot;
    const uint8_t *top, *bottom;  // next item to ask for: this lane's bytes of rows g and g + 8
    int left, room;               // items not asked for yet, in all and of the tile
};

template <typename Open>
__device__ __forceinline__ void w8_issue(W8Ring& r, uint32_t slot, int items, Open&& open) {
    if (r.left > 0) {
        const uint32_t to = r.base + slot;
        w8_copy(to, r.top);
        w8_copy(to + 512, r.bottom);
        w8_copy(to + 1024, r.top + 64);
        w8_copy(to + 1536, r.bottom + 64);
        r.top += 128;
        r.bottom += 128;
        --r.left;
        if (--r.room == 0 && r.left > 0) {
            open();
            r.room = items;
        }
    }
    w8_commit();
}

struct W8Block {
    int expert, row0, count;
};

template <bool SELF>
__device__ __forceinline__ W8Block w8_block(const W8Params& p, const W8Plan& plan, int b) {
    W8Block k;
    if (SELF) {
        k.expert = plan.expert[b];
        k.row0 = plan.row0[b];
        k.count = plan.count[b];
    } else {
        const GroupBlock g = p.blocks[b];
        k.expert = g.key;
        k.row0 = g.first;
        k.count = g.count;
    }
    return k;
}

// ------------------------------------------------------------------------------------------------ spans of whole tiles (gate_up; down, general form)
template <typename T, bool BLOCK, bool SELF, bool DOWN>
__global__ void __launch_bounds__(kW8Threads, 2) moe_w8_tiles_kernel(const __grid_constant__ W8Params p) {
    constexpr int kSubs = DOWN ? 2 : 1;  // rows 0 .. 3 and 4 .. 7 of a block, each as value and remainder; or its eight rows as they are
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, j = lane & 3;
    float4* part = reinterpret_cast<float4*>(smem + kW8Warps * kW8Depth * kW8Item);  // [warps][first, last tile][kSubs][32]
    W8Plan& plan = *reinterpret_cast<W8Plan*>(part + kW8Warps * 2 * kSubs * 32);

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // behind the wait: what follows may read this launch's inputs early
    if (SELF) w8_plan(p, plan);
    const int n_blocks = SELF ? plan.n_blocks : *p.n_blocks;
    const int K = DOWN ? p.I : p.H, items = K / 128;
    const int tiles = DOWN ? p.H / 16 : p.I / 8;  // of a block
    const int64_t units = static_cast<int64_t>(n_blocks) * tiles;
    const int64_t u0 = units * blockIdx.x / gridDim.x;
    const int span = static_cast<int>(units * (blockIdx.x + 1) / gridDim.x - u0);
    const int64_t total = static_cast<int64_t>(span) * items;
    auto share = [&](int w) { return total * w / kW8Warps; };
    const int64_t q0 = share(warp);
    const int n = static_cast<int>(share(warp + 1) - q0);
    const int first = static_cast<int>(q0 / items), skip = static_cast<int>(q0 - static_cast<int64_t>(first) * items);

    // tile `rel` of the span: block, channels, this lane's two rows of weights
    auto block_of = [&](int rel) { return static_cast<int>((u0 + rel) / tiles); };
    auto rows_of = [&](int rel, int k, const uint8_t*& top, const uint8_t*& bottom, int& expert, int& chan) {
        const int b = block_of(rel);
        chan = static_cast<int>(u0 + rel - static_cast<int64_t>(b) * tiles);
        expert = w8_block<SELF>(p, plan, b).expert;
        const int rows = DOWN ? p.H : 2 * p.I;
        const int r0 = DOWN ? chan * 16 + g : chan * 8 + g;
        top = p.w + (static_cast<size_t>(expert) * rows + r0) * K + k * 128 + 16 * j;
        bottom = top + static_cast<size_t>(DOWN ? 8 : p.I) * K;
    };
    W8Ring ring;
    ring.base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (kW8Depth * kW8Item) + lane * 16;
    ring.left = n;
    int ask = first;  // tile of the next item to ask for
    int unused_e, unused_c;
    if (n > 0) rows_of(ask, skip, ring.top, ring.bottom, unused_e, unused_c);
    ring.room = items - skip;
    auto open = [&]() {
        ++ask;
        rows_of(ask, 0, ring.top, ring.bottom, unused_e, unused_c);
    };
#pragma unroll 1
    for (int d = 0; d < kW8Depth; ++d) w8_issue(ring, d * kW8Item, items, open);

    // what a lane reads beside the weights, one item ahead: its column of the rows, the block's scales
    uint4 next[kSubs][4];
    float next_s0 = 1.f, next_s1 = 1.f;
    int at = first, k_at = skip;   // the item that `next` holds
    const T *col[kSubs];           // this lane's column of the tile that `next` is of
    const float *s0 = nullptr, *s1 = nullptr;
    auto enter = [&]() {           // a new tile
        const W8Block blk = w8_block<SELF>(p, plan, block_of(at));
        const int chan = static_cast<int>(u0 + at - static_cast<int64_t>(block_of(at)) * tiles);
#pragma unroll
        for (int s = 0; s < kSubs; ++s) {
            if (DOWN) {
                const int r = 4 * s + (g & 3);
                col[s] = r < blk.count ? static_cast<const T*>(g < 4 ? p.hi : p.lo) + static_cast<size_t>(blk.row0 + r) * K + 16 * j : nullptr;
            } else {
                int token = 0;
                if (g < blk.count) token = SELF ? plan.token[blk.row0 + g] : p.rows[blk.row0 + g] / p.topk;
                col[s] = g < blk.count ? static_cast<const T*>(p.x) + static_cast<size_t>(token) * K + 16 * j : nullptr;
            }
        }
        if (BLOCK) {
            const int rows = (DOWN ? p.H : 2 * p.I) / 128;
            s0 = p.scale + (static_cast<size_t>(blk.expert) * rows + (DOWN ? chan / 8 : chan / 16)) * items;
            s1 = DOWN ? s0 : s0 + static_cast<size_t>(p.I / 128) * items;
        } else {
            s0 = p.scale + static_cast<size_t>(blk.expert) * (DOWN ? p.H : 2 * p.I) + (DOWN ? chan * 16 + g : chan * 8 + g);
            s1 = s0 + (DOWN ? 8 : p.I);
        }
    };
    auto fetch = [&]() {
#pragma unroll
        for (int s = 0; s < kSubs; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                next[s][i] = col[s] ? (DOWN ? __ldcg(reinterpret_cast<const uint4*>(col[s] + k_at * 128 + (i >> 1) * 64 + (i & 1) * 8)) : *reinterpret_cast<const uint4*>(col[s] + k_at * 128 + (i >> 1) * 64 + (i & 1) * 8)) : make_uint4(0, 0, 0, 0);
        if (BLOCK) {
            next_s0 = __ldg(s0 + k_at);
            next_s1 = __ldg(s1 + k_at);
        } else {
            next_s0 = __ldg(s0);
            next_s1 = __ldg(s1);
        }
    };
    // the finished sums of a tile (lane: channels g and g + 8, or gate and up of channel g; columns 2 j, 2 j + 1)
    auto finish = [&](int rel, float (&sum)[kSubs][4]) {
        const int b = block_of(rel);
        const W8Block blk = w8_block<SELF>(p, plan, b);
        const int chan = static_cast<int>(u0 + rel - static_cast<int64_t>(b) * tiles);
        if (!DOWN) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 2 * j + i;
                if (r >= blk.count) continue;
                const float gate = sum[0][i], up = sum[0][2 + i];
                T hi, lo;
                split16<T>(gate / (1.f + expf(-gate)) * up, hi, lo);
                const size_t to = static_cast<size_t>(blk.row0 + r) * p.I + chan * 8 + g;
                static_cast<T*>(p.hi)[to] = hi;
                static_cast<T*>(p.lo)[to] = lo;
            }
        } else {
#pragma unroll
            for (int s = 0; s < kSubs; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = sum[s][i] + __shfl_xor_sync(0xFFFFFFFFu, sum[s][i], 2);  // value + remainder: columns r and r + 4
                    const int r = 4 * s + 2 * j + (i & 1);
                    if (j < 2 && r < blk.count) p.rows_out[static_cast<size_t>(p.rows[blk.row0 + r]) * p.H + chan * 16 + g + 8 * (i >> 1)] = v;
                }
        }
    };

    if (n > 0) {
        enter();
        fetch();
    }
    int slot = 0;
    int rel = first, it = skip;
    for (int i = 0; i < n;) {
        const int stretch = min(items - it, n - i);
        float sum[kSubs][4];
#pragma unroll
        for (int s = 0; s < kSubs; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[s][e] = 0.f;
        for (int c = 0; c < stretch; ++c) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kW8Depth - 1) : "memory");
            uint4 now[kSubs][4];
#pragma unroll
            for (int s = 0; s < kSubs; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) now[s][e] = next[s][e];
            const float f0 = next_s0, f1 = next_s1;
            if (i + c + 1 < n) {
                if (++k_at == items) {
                    k_at = 0;
                    ++at;
                    enter();
                }
                fetch();
            }
            float acc[kSubs][4];
#pragma unroll
            for (int s = 0; s < kSubs; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[s][e] = 0.f;
            w8_item<T, kSubs>(ring.base + slot, now, acc);
            w8_issue(ring, slot, items, open);
            slot = slot + kW8Item == kW8Depth * kW8Item ? 0 : slot + kW8Item;
#pragma unroll
            for (int s = 0; s < kSubs; ++s) {
                sum[s][0] = fmaf(acc[s][0], f0, sum[s][0]);
                sum[s][1] = fmaf(acc[s][1], f0, sum[s][1]);
                sum[s][2] = fmaf(acc[s][2], f1, sum[s][2]);
                sum[s][3] = fmaf(acc[s][3], f1, sum[s][3]);
            }
        }
        if (stretch == items) {
            finish(rel, sum);
        } else {  // a tile that another warp has a part of
#pragma unroll
            for (int s = 0; s < kSubs; ++s)
                part[((warp * 2 + (rel == first ? 0 : 1)) * kSubs + s) * 32 + lane] = make_float4(sum[s][0], sum[s][1], sum[s][2], sum[s][3]);
        }
        i += stretch;
        it = 0;
        ++rel;
    }
    __syncthreads();
    // the shared tiles, in the order of the warps that have a part
    for (int t = warp; t < span; t += kW8Warps) {
        const int64_t lo_item = static_cast<int64_t>(t) * items, hi_item = lo_item + items;
        float sum[kSubs][4];
#pragma unroll
        for (int s = 0; s < kSubs; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[s][e] = 0.f;
        int parts = 0;
        bool whole = false;
        for (int w = 0; w < kW8Warps; ++w) {
            const int64_t a = share(w), b = share(w + 1);
            if (a >= hi_item || b <= lo_item || a == b) continue;
            if (a <= lo_item && b >= hi_item) {
                whole = true;
                break;
            }
            ++parts;
            const int which = static_cast<int>(a / items) == t ? 0 : 1;
#pragma unroll
            for (int s = 0; s < kSubs; ++s) {
                const float4 v = part[((w * 2 + which) * kSubs + s) * 32 + lane];
                sum[s][0] += v.x;
                sum[s][1] += v.y;
                sum[s][2] += v.z;
                sum[s][3] += v.w;
            }
        }
        if (!whole && parts) finish(t, sum);
    }
}

// ------------------------------------------------------------------------------------------------ down, sixteen channels of all blocks
template <typename T, bool BLOCK>
__global__ void __launch_bounds__(kW8Threads, 2) moe_w8_down_kernel(const __grid_constant__ W8Params p) {
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, j = lane & 3;
    float* sums = reinterpret_cast<float*>(smem + kW8Warps * kW8Depth * kW8Item);  // [warps][T][16]
    W8Plan& plan = *reinterpret_cast<W8Plan*>(sums + kW8Warps * p.T * 16);
    // The launch before this one waited for what came before it ahead of letting this one start, so the logits may be read here and the
    // weights asked for; what it computes is read behind the wait.
    w8_plan(p, plan);
    for (int i = tid; i < kW8Warps * p.T * 16; i += kW8Threads) sums[i] = 0.f;
    __syncthreads();
    const int items = p.I / 128, chan = blockIdx.x * 16;
    const int total = plan.n_blocks * items;
    const int q0 = total * warp / kW8Warps, n = total * (warp + 1) / kW8Warps - q0;
    const int first = q0 / items, skip = q0 - first * items;
    W8Ring ring;
    ring.base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (kW8Depth * kW8Item) + lane * 16;
    ring.left = n;
    ring.room = items - skip;
    int ask = first;
    auto rows_of = [&](int b, int k) {
        ring.top = p.w + (static_cast<size_t>(plan.expert[b]) * p.H + chan + g) * p.I + k * 128 + 16 * j;
        ring.bottom = ring.top + static_cast<size_t>(8) * p.I;
    };
    if (n > 0) rows_of(ask, skip);
    auto open = [&]() { rows_of(++ask, 0); };
#pragma unroll 1
    for (int d = 0; d < kW8Depth; ++d) w8_issue(ring, d * kW8Item, items, open);

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    uint4 next[2][4];
    float next_s0 = 1.f, next_s1 = 1.f;
    int at = first, k_at = skip;
    const T* col[2];
    const float *s0 = nullptr, *s1 = nullptr;
    auto enter = [&]() {
        const int row0 = plan.row0[at], count = plan.count[at], expert = plan.expert[at];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int r = 4 * s + (g & 3);
            col[s] = r < count ? static_cast<const T*>(g < 4 ? p.hi : p.lo) + static_cast<size_t>(row0 + r) * p.I + 16 * j : nullptr;
        }
        if (BLOCK) {
            s0 = s1 = p.scale + (static_cast<size_t>(expert) * (p.H / 128) + chan / 128) * items;
        } else {
            s0 = p.scale + static_cast<size_t>(expert) * p.H + chan + g;
            s1 = s0 + 8;
        }
    };
    auto fetch = [&]() {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                next[s][i] = col[s] ? __ldcg(reinterpret_cast<const uint4*>(col[s] + k_at * 128 + (i >> 1) * 64 + (i & 1) * 8)) : make_uint4(0, 0, 0, 0);
        next_s0 = __ldg(BLOCK ? s0 + k_at : s0);
        next_s1 = __ldg(BLOCK ? s1 + k_at : s1);
    };
    if (n > 0) {
        enter();
        fetch();
    }
    float* mine = sums + warp * p.T * 16;
    int slot = 0, rel = first, it = skip;
    for (int i = 0; i < n;) {
        const int stretch = min(items - it, n - i);
        float sum[2][4];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[s][e] = 0.f;
        for (int c = 0; c < stretch; ++c) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kW8Depth - 1) : "memory");
            uint4 now[2][4];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) now[s][e] = next[s][e];
            const float f0 = next_s0, f1 = next_s1;
            if (i + c + 1 < n) {
                if (++k_at == items) {
                    k_at = 0;
                    ++at;
                    enter();
                }
                fetch();
            }
            float acc[2][4];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[s][e] = 0.f;
            w8_item<T, 2>(ring.base + slot, now, acc);
            w8_issue(ring, slot, items, open);
            slot = slot + kW8Item == kW8Depth * kW8Item ? 0 : slot + kW8Item;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                sum[s][0] = fmaf(acc[s][0], f0, sum[s][0]);
                sum[s][1] = fmaf(acc[s][1], f0, sum[s][1]);
                sum[s][2] = fmaf(acc[s][2], f1, sum[s][2]);
                sum[s][3] = fmaf(acc[s][3], f1, sum[s][3]);
            }
        }
        // this warp's part of the block's rows, weighted, to its tokens' sums (the rows of a block are different tokens)
        const int row0 = plan.row0[rel], count = plan.count[rel];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = sum[s][e] + __shfl_xor_sync(0xFFFFFFFFu, sum[s][e], 2);
                const int r = 4 * s + 2 * j + (e & 1);
                if (j < 2 && r < count) mine[plan.token[row0 + r] * 16 + g + 8 * (e >> 1)] += plan.score[row0 + r] * v;
            }
        __syncwarp();
        i += stretch;
        it = 0;
        ++rel;
    }
    __syncthreads();
    for (int i = tid; i < p.T * 16; i += kW8Threads) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kW8Warps; ++w) v += sums[w * p.T * 16 + i];
        static_cast<T*>(p.y)[static_cast<size_t>(i >> 4) * p.H + chan + (i & 15)] = from_float<T>(v);
    }
}

// y[t] = sum_j score[t, j] rows[t topk + j], four channels a thread, picks in ascending expert order.
template <typename T>
__global__ void __launch_bounds__(256) moe_w8_combine_kernel(const float4* __restrict__ rows, const float* __restrict__ scores, int64_t vecs, int row_vecs, int topk,
                                                             T* __restrict__ y) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t i = blockIdx.x * int64_t(256) + threadIdx.x;
    if (i >= vecs) return;
    const int64_t t = i / row_vecs, v = i - t * row_vecs;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < topk; ++k) {
        const float p = scores[t * topk + k];
        const float4 r = __ldcg(rows + (t * topk + k) * row_vecs + v);
        s.x = fmaf(p, r.x, s.x);
        s.y = fmaf(p, r.y, s.y);
        s.z = fmaf(p, r.z, s.z);
        s.w = fmaf(p, r.w, s.w);
    }
    T* to = y + i * 4;
    to[0] = from_float<T>(s.x);
    to[1] = from_float<T>(s.y);
    to[2] = from_float<T>(s.z);
    to[3] = from_float<T>(s.w);
}

// ------------------------------------------------------------------------------------------------ host
static size_t w8_align(size_t v) { return (v + 255) / 256 * 256; }

struct W8Workspace {
    void *hi, *lo;
    int32_t *ids, *rows, *n_blocks;
    float *scores, *rows_out;
    GroupBlock* blocks;
    size_t bytes;
};

static bool w8_self(int64_t T, int64_t E) { return T <= kW8SelfTokens && E <= kW8SelfExperts; }

static W8Workspace w8_carve(void* base, int64_t T, int64_t E, int64_t topk, int64_t H, int64_t I) {
    W8Workspace w = {};
    unsigned char* b = static_cast<unsigned char*>(base);
    size_t o = 0;
    auto take = [&](size_t bytes) {
        void* at = b + o;
        o += w8_align(bytes);
        return at;
    };
    const int64_t R = T * topk;
    w.hi = take(static_cast<size_t>(R) * I * 2);
    w.lo = take(static_cast<size_t>(R) * I * 2);
    if (!w8_self(T, E)) {
        w.ids = static_cast<int32_t*>(take(R * 4));
        w.scores = static_cast<float*>(take(R * 4));
        w.rows = static_cast<int32_t*>(take(R * 4));
        w.n_blocks = static_cast<int32_t*>(take(4));
        w.blocks = static_cast<GroupBlock*>(take(static_cast<size_t>(group_max_blocks(R, E, kW8BlockRows, false)) * sizeof(GroupBlock)));
        w.rows_out = static_cast<float*>(take(static_cast<size_t>(R) * H * 4));
    }
    w.bytes = o;
    return w;
}

template <typename Kernel, typename... A>
static int w8_launch(Kernel kernel, int64_t grid, size_t smem, cudaStream_t stream, A... args) {
    EQ_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 113 * 1024));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kW8Threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    EQ_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, args...));
    return EQ_OK;
}

template <typename T, bool BLOCK>
static int w8_forward(W8Params p, const uint8_t* gate_up, const float* gate_up_scale, const uint8_t* down, const float* down_scale, const W8Workspace& w,
                      cudaStream_t stream) {
    const size_t ring = static_cast<size_t>(kW8Warps) * kW8Depth * kW8Item;
    const size_t part = kW8Warps * 2 * 32 * sizeof(float4);
    p.w = gate_up;
    p.scale = gate_up_scale;
    const int64_t R = static_cast<int64_t>(p.T) * p.topk;
    if (w8_self(p.T, p.E)) {
        const int64_t tiles = R * (p.I / 8);
        int st = w8_launch(moe_w8_tiles_kernel<T, BLOCK, true, false>, tiles < sm_count() ? tiles : sm_count(), ring + part + sizeof(W8Plan), stream, p);
        if (st != EQ_OK) return st;
        p.w = down;
        p.scale = down_scale;
        return w8_launch(moe_w8_down_kernel<T, BLOCK>, p.H / 16, ring + static_cast<size_t>(kW8Warps) * p.T * 16 * sizeof(float) + sizeof(W8Plan), stream, p);
    }
    int st = eq_moe_route(p.logits, p.T, p.E, p.topk, 1, w.ids, w.scores, stream);
    if (st != EQ_OK) return st;
    st = group_rows_launch(w.ids, static_cast<int>(R), p.E, false, kW8BlockRows, false, w.blocks, w.n_blocks, w.rows, nullptr, stream);
    if (st != EQ_OK) return st;
    st = w8_launch(moe_w8_tiles_kernel<T, BLOCK, false, false>, 2 * sm_count(), ring + part, stream, p);
    if (st != EQ_OK) return st;
    p.w = down;
    p.scale = down_scale;
    st = w8_launch(moe_w8_tiles_kernel<T, BLOCK, false, true>, 2 * sm_count(), ring + 2 * part, stream, p);
    if (st != EQ_OK) return st;
    const int64_t vecs = static_cast<int64_t>(p.T) * p.H / 4;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ceil_div(vecs, 256)));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    EQ_CUDA_OK(cudaLaunchKernelEx(&cfg, moe_w8_combine_kernel<T>, reinterpret_cast<const float4*>(w.rows_out), static_cast<const float*>(w.scores), vecs, p.H / 4, p.topk,
                                  static_cast<T*>(p.y)));
    return EQ_OK;
}

}  // namespace eq

using namespace eq;

extern "C" size_t eq_moe_w8a16_workspace_bytes(int64_t T, int64_t E, int64_t topk, int64_t H, int64_t I) {
    if (T <= 0 || E <= 0 || topk <= 0 || H <= 0 || I <= 0) return 0;
    return w8_carve(nullptr, T, E, topk, H, I).bytes;
}

extern "C" int eq_moe_w8a16(const uint8_t* gate_up, const float* gate_up_scale, const uint8_t* down, const float* down_scale, int block_scales, int64_t E,
                            int64_t topk, int64_t H, int64_t I, const void* x, const float* router_logits, int64_t T, int act_dtype, void* y, void* workspace,
                            size_t workspace_bytes, void* stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    EQ_REQUIRE(T >= 0 && E > 0 && topk > 0 && H > 0 && I > 0, EQ_ERR_BAD_ARG, "eq_moe_w8a16: bad extents T=%lld E=%lld topk=%lld H=%lld I=%lld", (long long)T, (long long)E,
               (long long)topk, (long long)H, (long long)I);
    EQ_REQUIRE(block_scales == 0 || block_scales == 1, EQ_ERR_BAD_ARG, "eq_moe_w8a16: block_scales is 0 (per output channel) or 1 (128 x 128 blocks)");
    EQ_REQUIRE(act_dtype == EQ_F16 || act_dtype == EQ_BF16, EQ_ERR_BAD_ARG, "eq_moe_w8a16: activations must be f16 or bf16");
    EQ_REQUIRE(E <= 1024 && topk <= kW8MaxTopK && topk <= E, EQ_ERR_UNSUPPORTED, "eq_moe_w8a16: needs 0 < top-k <= 16 and E <= 1024");
    EQ_REQUIRE(H % 128 == 0 && I % 128 == 0 && H < (1 << 24) && I < (1 << 24), EQ_ERR_UNSUPPORTED, "eq_moe_w8a16: needs hidden and intermediate sizes that are multiples of 128");
    EQ_REQUIRE(T < (1 << 24), EQ_ERR_UNSUPPORTED, "eq_moe_w8a16: too many tokens");
    if (T == 0) return EQ_OK;
    EQ_REQUIRE(gate_up && gate_up_scale && down && down_scale && x && router_logits && y, EQ_ERR_BAD_ARG, "eq_moe_w8a16: null pointer");
    EQ_REQUIRE(aligned(gate_up, 16) && aligned(down, 16) && aligned(x, 16) && aligned(y, 16), EQ_ERR_BAD_ALIGN, "eq_moe_w8a16: weights and activations must be 16-byte aligned");
    EQ_REQUIRE(aligned(gate_up_scale, 4) && aligned(down_scale, 4) && aligned(router_logits, 4), EQ_ERR_BAD_ALIGN, "eq_moe_w8a16: scales and logits must be 4-byte aligned");
    const size_t need = eq_moe_w8a16_workspace_bytes(T, E, topk, H, I);
    EQ_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= need, EQ_ERR_WORKSPACE, "eq_moe_w8a16: workspace of %zu bytes (256-byte aligned) needed, %zu given",
               need, workspace_bytes);
    const W8Workspace w = w8_carve(workspace, T, E, topk, H, I);
    W8Params p = {};
    p.logits = router_logits;
    p.x = x;
    p.hi = w.hi;
    p.lo = w.lo;
    p.y = y;
    p.rows_out = w.rows_out;
    p.blocks = w.blocks;
    p.n_blocks = w.n_blocks;
    p.rows = w.rows;
    p.T = static_cast<int>(T);
    p.E = static_cast<int>(E);
    p.topk = static_cast<int>(topk);
    p.H = static_cast<int>(H);
    p.I = static_cast<int>(I);
    if (act_dtype == EQ_F16)
        return block_scales ? w8_forward<__half, true>(p, gate_up, gate_up_scale, down, down_scale, w, stream)
                            : w8_forward<__half, false>(p, gate_up, gate_up_scale, down, down_scale, w, stream);
    return block_scales ? w8_forward<__nv_bfloat16, true>(p, gate_up, gate_up_scale, down, down_scale, w, stream)
                        : w8_forward<__nv_bfloat16, false>(p, gate_up, gate_up_scale, down, down_scale, w, stream);
}
