// Routed MoE layer of a few tokens on FP8 (e4m3) experts, weights as the checkpoint stores them:
//     y[t] = sum_j p[t, j] W_down[e] (silu(W_gate[e] x[t]) * (W_up[e] x[t])),  e = id[t, j],
// id the topk experts of largest router logit (ties to the lowest id), p their softmax, renormalised over the picks.
//
// A weight is bits x scale, the scale per output channel or per 128 x 128 block, applied to f32 sums.  e4m3 is a part of f16, so a weight is expanded
// to f16 by one conversion a pair, exactly, whatever the activations' type, and these are brought to f16 without loss: a row of bf16 is multiplied by a power of
// two that takes its largest value to [2^14, 2^15) (its eight bits are exact in f16 down to 2^-31 of that, and off by 2^-39 of it below); a row of silu(gate) * up,
// in f32, the same way, as two numbers, value and remainder (2^-22 of itself, 2^-39 of the largest).  Products are mma.sync m16n8k16 with f32 sums.  The layer
// rounds once, as y is stored.  (16 tokens of 128 experts of 2048 x 768 take 87 us a layer.  bf16 MMAs want two conversions and a packing more a pair, 264
// instructions per 2 KB of weights beside the 89 cycles that HBM needs for them: 123 us.  m16n8k32 on e4m3 parts of the activations converts both
// operands inside every MMA: 189 us.)
//
// What bounds it: the bytes of the picked experts, as long as few rows share one.  5 tokens of 8 experts of 4096 x 14336 stream them at 5.0 to 5.2 TB/s (five of them
// picked 176 us, seven 242),
// 16 tokens as above at 4.5 beside routing, the seam of the two products and their ends; one token (38 MB, 17.6 us, 5.8 at the rate of HBM) is a chain of latencies,
// of which routing takes 2.8 us, the seam with the split of silu * up 2 and each product 4.  With more rows the MMAs' operands: 200 tokens 189 us for 93 of bytes.
//
// Up to 32 tokens and 256 experts:
//   gate_up  Every CTA groups the picks by expert itself: a block is at most eight rows (picks) of one expert, so
//            an expert that several tokens picked is read once.  The blocks' tiles of eight gate and the same eight up rows (one MMA
//            A operand of sixteen rows) are one stream, cut into equal spans over the CTAs and in a CTA into equal shares of 128-element items over its
//            warps.  A tile's silu and product happen in the registers of whoever has its sums; tiles that several warps share meet in shared
//            memory in warp order.
//   down     A cluster of CTAs has sixteen output channels of ALL the blocks: the picks of a token meet inside it (f32, a fixed order), y is written
//            once, and nothing is combined in memory.  It has grouped the picks and asked for its first weights before the launch ahead of it ends.
// Where a CTA of either launch fits an SM with f16 activations of its own (w8_form) these two launches are the layer, one CTA an SM each, so that the second
// one is resident, has routed too and asked for its first weights while the first one runs.  Else w8_prep_kernel routes the tokens and brings x (of bf16) to f16 ahead of them.
// Then no launch has to come between the two: the rows' largest values are found as they are written, and the second one splits what it reads of them.
// Above, w8_prep_kernel and group.cu list the blocks, w8_parts_kernel splits the rows of silu * up (there are so many CTAs for each row that they would do it
// many times: 64 tokens of 128 experts of 2048 x 768 152 us for 143), and both products run as streams of tiles; the down rows go to memory in f32 and
// moe_w8_combine_kernel adds them.
//
// Weights reach a lane through a ring in shared memory that the lane fills by cp.async for itself (16 bytes of a row: K indices 16 j .. 16 j + 15
// of each half of the item, in both operands alike), the scales beside them, so no warp waits for another.  mma.sync and not tcgen05: with at most eight rows the weights'
// bytes bound the layer.
#include <type_traits>

#include "group.cuh"
#include "mma_sync.cuh"

namespace eq {

constexpr int kW8Threads = 256;
constexpr int kW8Warps = kW8Threads / 32;
// A warp's items are MW x 16 rows x 128 elements, in a ring of w8_depth(MW).
// With one CTA of either launch on an SM (few) it is deeper, half of what a warp reads asked for at once: a token of 128 experts of 2048 x 768 21.2 us with
// three, 17.8 with five.  (Four and six: the two no longer fit one SM, 21.3.)
constexpr int w8_depth(int mw, bool few) { return few ? 5 : mw == 1 ? 3 : 2; }
constexpr int w8_ring(int mw, bool few) { return w8_depth(mw, few) * mw * 2048; }
// Their scales come with them: of sixteen rows eight pairs (rows g, g + 8), of a 128 x 128 block's rows all alike.
constexpr int w8_scales(int mw, bool block) { return 64 * (block ? 1 : mw); }
constexpr int w8_stage(int mw, bool few, bool block) { return w8_depth(mw, few) * w8_scales(mw, block); }
constexpr int kW8SelfTokens = 32;       // tokens up to which the CTAs group the picks themselves (one bit each of a word)
constexpr int kW8SelfExperts = 256;
constexpr int kW8MaxTopK = 16;
constexpr int kW8SelfPicks = kW8SelfTokens * kW8MaxTopK;
constexpr int kW8BlockRows = 8;
constexpr int kW8PartsH = 2;            // value and remainder of silu(gate) * up

struct W8Params {
    const uint8_t* w;         // this phase's weights: gate_up [E][2I][H] or down [E][H][I]
    const float* scale;       // [E][2I] / [E][H], or [E][2I / 128][H / 128] / [E][H / 128][I / 128]
    const float* logits;      // [T][E]
    const void* x;            // [T][H]
    const int32_t* ids;       // [T][topk] -1: dropped; null: the CTAs route
    const float* shares;      // [T][topk]
    const __half* x16;        // [T][H] x in f16, where the CTAs do not make it
    const float* x_scale;     // [T] what brings it back; null: nothing does
    float* h;                 // [picks][I] silu(gate) * up, in expert order
    uint32_t* h_max;          // [picks] bits of a row's largest finite magnitude; null: nobody reads them
    const __half* h16;        // [picks][2][I] and what brings it back, general form
    const float* h_scale;
    void* y;                  // [T][H]
    float* rows_out;          // [picks][H], general form
    const GroupBlock* blocks; // general form
    const int32_t* n_blocks;
    const int32_t* rows;      // pick of each row in expert order
    int T, E, topk, H, I;
};

// ------------------------------------------------------------------------------------------------ routing and grouping
// The picks in expert order, worked out by a CTA for itself.
struct W8Plan {
    uint32_t tokens[kW8SelfExperts];      // tokens that picked an expert
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

// One warp, one token of at most 32 NV experts: picks in the order of their logits and their shares to store(place, id, share); -1: no such pick.
template <int NV, typename Store>
__device__ __forceinline__ void w8_route(const float* __restrict__ logits, int E, int topk, Store&& store) {
    const int lane = threadIdx.x & 31;
    uint32_t key[NV];
    bool nan = false;
#pragma unroll
    for (int b = 0; b < NV; ++b) {
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
        for (int b = 0; b < NV; ++b)
            if (key[b] > best) {
                best = key[b];
                at = b;
            }
        const uint32_t win = __reduce_max_sync(0xFFFFFFFFu, best);
        const uint32_t e = __reduce_min_sync(0xFFFFFFFFu, best == win && win ? static_cast<uint32_t>(lane + 32 * at) : 0xFFFFFFFFu);
        if (win && e == static_cast<uint32_t>(lane + 32 * at)) {
#pragma unroll
            for (int b = 0; b < NV; ++b)
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
    if (lane < topk) store(lane, my_id, nan ? __int_as_float(0x7FC00000) : p / sum);  // the softmax of a row that holds a NaN
}

// The picks of all tokens: read, or routed by warps 0 .. warps - 1.  No barrier.
__device__ __forceinline__ void w8_picks(const W8Params& p, W8Plan& plan, int warps) {
    const int tid = threadIdx.x, warp = tid >> 5;
    if (p.ids) {
        for (int i = tid; i < p.T * p.topk; i += kW8Threads) {
            plan.id[i] = static_cast<int16_t>(__ldcg(p.ids + i));
            plan.share[i] = __ldcg(p.shares + i);
        }
    } else if (warp < warps) {
        for (int t = warp; t < p.T; t += warps)
            w8_route<kW8SelfExperts / 32>(p.logits + static_cast<size_t>(t) * p.E, p.E, p.topk, [&](int k, int id, float share) {
                plan.id[t * p.topk + k] = static_cast<int16_t>(id);
                plan.share[t * p.topk + k] = share;
            });
    }
}
// The blocks, from the picks.  Begins and ends with a barrier.
__device__ __forceinline__ void w8_group(const W8Params& p, W8Plan& plan) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, picks = p.T * p.topk;
    static_assert(kW8SelfExperts == kW8Threads, "an expert a thread");
    if (p.T == 1) {  // every pick is a block
        __syncthreads();
        if (tid < 32) {
            const int e = tid < picks ? plan.id[tid] : -1;
            if (e >= 0) {  // (no such pick: none behind it either)
                plan.expert[tid] = static_cast<uint16_t>(e);
                plan.row0[tid] = static_cast<uint16_t>(tid);
                plan.count[tid] = 1;
                plan.token[tid] = 0;
                plan.score[tid] = plan.share[tid];
            }
            const uint32_t real = __ballot_sync(0xFFFFFFFFu, e >= 0);
            if (tid == 0) plan.n_blocks = __popc(real);
        }
        __syncthreads();
        return;
    }
    plan.tokens[tid] = 0;
    __syncthreads();
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

// ------------------------------------------------------------------------------------------------ activations in f16
// The power of two that brings a largest value of `big` to [2^14, 2^15); 1 for zero.
__device__ __forceinline__ float w8_up(float big) {
    const int e = static_cast<int>(__float_as_uint(big) >> 23);  // biased; big >= 0
    return big > 0.f ? __uint_as_float(static_cast<uint32_t>(min(254, 127 + 14 - (e - 127))) << 23) : 1.f;
}
// Value and, where P is 2, remainder of two neighbouring values.  What is not finite has no remainder.
template <int P>
__device__ __forceinline__ void w8_split(float v0, float v1, uint32_t (&out)[P]) {
    const __half2 hi = __floats2half2_rn(v0, v1);
    out[0] = *reinterpret_cast<const uint32_t*>(&hi);
    if (P == 2) {
        const float2 back = __half22float2(hi);
        const __half2 lo = __floats2half2_rn(fabsf(v0) < INFINITY ? v0 - back.x : 0.f, fabsf(v1) < INFINITY ? v1 - back.y : 0.f);
        out[P - 1] = *reinterpret_cast<const uint32_t*>(&lo);
    }
}
// Four neighbouring values of a row.
template <typename InT>
__device__ __forceinline__ float4 w8_load4(const InT* p) {
    if constexpr (std::is_same<InT, float>::value) {
        return __ldcg(reinterpret_cast<const float4*>(p));
    } else {
        const uint2 raw = __ldcg(reinterpret_cast<const uint2*>(p));
        const InT* e = reinterpret_cast<const InT*>(&raw);
        return make_float4(to_float(e[0]), to_float(e[1]), to_float(e[2]), to_float(e[3]));
    }
}
__device__ __forceinline__ float w8_warp_max(float v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, off));
    return v;
}
// Rows 0 .. count - 1 of n values (a multiple of 128) brought to f16 by `warps` warps (all 8, or 4), of which this is number `warp`: parts to
// put(row, part, index, four f16), the power of two that brings a row's parts back to done(row, it).  A row is taken by as many of them as there are for it; a
// lane's first eight loads are in flight together and are not read again.
template <int P, typename InT, typename Put, typename Done>
__device__ __forceinline__ void w8_rows_parts(const InT* rows, int count, int n, int warp, int warps, Put&& put, Done&& done) {
    constexpr int kHeld = 8;
    __shared__ float warps_max[kW8Warps];
    const int lane = threadIdx.x & 31;
    int wide = warps;
    while (wide > 1 && wide * count > warps) wide /= 2;
    const int at_once = warps / wide;
    auto meet = [&]() {
        if (warps == kW8Warps) __syncthreads();
        else asm volatile("bar.sync 1, 128;" ::: "memory");
    };
    const int at = 4 * ((warp % wide) * 32 + lane), stride = 4 * 32 * wide;
    for (int row0 = 0; row0 < count; row0 += at_once) {
        const int row = row0 + warp / wide;
        const bool live = row < count;
        const InT* from = rows + static_cast<size_t>(live ? row : 0) * n;
        float4 held[kHeld];
        float big = 0.f;
        auto look = [&](const float4& v) {
            const float a[4] = {fabsf(v.x), fabsf(v.y), fabsf(v.z), fabsf(v.w)};
#pragma unroll
            for (int q = 0; q < 4; ++q) big = a[q] < INFINITY ? fmaxf(big, a[q]) : big;
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i) held[i] = live && at + i * stride < n ? w8_load4(from + at + i * stride) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) look(held[i]);
        if (live)
            for (int i = at + kHeld * stride; i < n; i += stride) look(w8_load4(from + i));
        big = w8_warp_max(big);
        if (wide > 1) {
            if (lane == 0) warps_max[warp] = big;
            meet();
            for (int w = 0; w < wide; ++w) big = fmaxf(big, warps_max[warp / wide * wide + w]);
        }
        const float up = w8_up(big);
        auto give = [&](const float4& v, int i) {
            uint32_t first[P], second[P];
            w8_split<P>(v.x * up, v.y * up, first);
            w8_split<P>(v.z * up, v.w * up, second);
#pragma unroll
            for (int p = 0; p < P; ++p) put(row, p, i, make_uint2(first[p], second[p]));
        };
        if (live) {
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (at + i * stride < n) give(held[i], at + i * stride);
            for (int i = at + kHeld * stride; i < n; i += stride) give(w8_load4(from + i), i);
            if (at == 0) done(row, 1.f / up);  // of a power of two: exact
        }
    }
}

// A CTA a token: its picks, a clear word for each of its rows of silu * up, and (x of bf16) its row in f16.
template <typename T, int NV>
__global__ void __launch_bounds__(kW8Threads) w8_prep_kernel(const __grid_constant__ W8Params p, int32_t* __restrict__ ids, float* __restrict__ shares,
                                                             __half* __restrict__ x16, float* __restrict__ x_scale) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // behind the wait: what follows may read this launch's inputs early
    const int t = blockIdx.x, warp = threadIdx.x >> 5;
    if (warp < 4) {
        if (warp == 0)
            w8_route<NV>(p.logits + static_cast<size_t>(t) * p.E, p.E, p.topk, [&](int k, int id, float share) {
                ids[static_cast<size_t>(t) * p.topk + k] = id;
                shares[static_cast<size_t>(t) * p.topk + k] = share;
                if (p.h_max) p.h_max[static_cast<size_t>(t) * p.topk + k] = 0u;
            });
    } else if constexpr (!std::is_same<T, __half>::value) {
        w8_rows_parts<1>(static_cast<const T*>(p.x) + static_cast<size_t>(t) * p.H, 1, p.H, warp - 4, 4,
                         [&](int, int, int i, uint2 four) { *reinterpret_cast<uint2*>(x16 + static_cast<size_t>(t) * p.H + i) = four; },
                         [&](int, float down) { x_scale[t] = down; });
    }
}

// A CTA a row of silu * up.
__global__ void __launch_bounds__(kW8Threads) w8_parts_kernel(const float* __restrict__ h, int n, __half* __restrict__ parts, float* __restrict__ scale) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __half* to = parts + static_cast<size_t>(blockIdx.x) * kW8PartsH * n;
    w8_rows_parts<kW8PartsH>(h + static_cast<size_t>(blockIdx.x) * n, 1, n, threadIdx.x >> 5, kW8Warps,
                             [&](int, int p, int i, uint2 four) { *reinterpret_cast<uint2*>(to + static_cast<size_t>(p) * n + i) = four; },
                             [&](int, float down) { scale[blockIdx.x] = down; });
}

// ------------------------------------------------------------------------------------------------ the stream of weights
__device__ __forceinline__ uint4 w8_lds(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
// Two e4m3 values (the low or the high half of a word) in f16.
__device__ __forceinline__ uint32_t w8_pair(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
    return h;
}
// One item, or with two groups of eight columns half of one: sum[c][m][16 rows][8 columns] += scale x W x over 128 or 64 elements, scale s0 for rows g and s1 for
// rows g + 8.  slot: this lane's first 16 bytes in the ring (of sixteen rows the first half of the elements, rows g; then rows g + 8; then the other
// half's); b: the lane's column of a group at the same K indices, sixteen values a half, of every part.
template <int P, int MW, int RB>
__device__ __forceinline__ void w8_item(uint32_t slot, const uint4 (&b)[RB][P][4 / RB], const float (&s0)[MW], const float (&s1)[MW], float (&sum)[RB][MW][4]) {
#pragma unroll
    for (int m = 0; m < MW; ++m) {
        float acc[2][4];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[c][e] = 0.f;
#pragma unroll
        for (int half = 0; half < 2 / RB; ++half) {
            const uint4 top = w8_lds(slot + m * 2048 + half * 1024), bottom = w8_lds(slot + m * 2048 + half * 1024 + 512);
            const uint32_t t[4] = {top.x, top.y, top.z, top.w}, u[4] = {bottom.x, bottom.y, bottom.z, bottom.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t a0 = w8_pair(t[q] & 0xFFFFu), a2 = w8_pair(t[q] >> 16), a1 = w8_pair(u[q] & 0xFFFFu), a3 = w8_pair(u[q] >> 16);
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                    for (int c = 0; c < RB; ++c) {  // two chains
                        const uint4& v = b[c][p][2 * half + (q >> 1)];
                        mma_16816<__half>(acc[RB == 2 ? c : P == 2 ? p : q & 1], a0, a1, a2, a3, q & 1 ? v.z : v.x, q & 1 ? v.w : v.y);
                    }
            }
        }
#pragma unroll
        for (int c = 0; c < RB; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[c][m][e] = fmaf(RB == 2 ? acc[c][e] : acc[0][e] + acc[1][e], e < 2 ? s0[m] : s1[m], sum[c][m][e]);
    }
}

__device__ __forceinline__ void w8_copy(uint32_t to, const uint8_t* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void w8_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// A warp's stream of items: tiles in order, each `items` items of 128 elements of K.  The owner says where a tile's rows lie for this lane.
struct W8Ring {
    uint32_t base;
    const uint8_t *top, *bottom;  // next item to ask for: this lane's bytes of rows g and g + 8
    int step;                     // bytes from sixteen rows to the next sixteen
    int left, room;               // items not asked for yet, in all and of the tile
    uint32_t scales;              // where this lane's rows' scales go
    const float *at0, *at1;       // theirs; per channel, those of the next sixteen rows `more` further
    int more;
};

__device__ __forceinline__ void w8_copy_scale(uint32_t to, const float* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

// The next item to stage `stage`.  (The lanes of a warp come here together: the scales are the one thing that they read from one another's copies.)
template <bool BLOCK, int MW, typename Open>
__device__ __forceinline__ void w8_issue(W8Ring& r, int stage, int items, Open&& open) {
    if (r.left > 0) {
        const uint32_t to = r.base + stage * MW * 2048;
#pragma unroll
        for (int m = 0; m < MW; ++m) {
            w8_copy(to + m * 2048, r.top + m * r.step);
            w8_copy(to + m * 2048 + 512, r.bottom + m * r.step);
            w8_copy(to + m * 2048 + 1024, r.top + m * r.step + 64);
            w8_copy(to + m * 2048 + 1536, r.bottom + m * r.step + 64);
        }
        if ((threadIdx.x & 3) == 0) {
#pragma unroll
            for (int m = 0; m < (BLOCK ? 1 : MW); ++m) {
                w8_copy_scale(r.scales + stage * w8_scales(MW, BLOCK) + m * 8, r.at0 + m * r.more);
                w8_copy_scale(r.scales + stage * w8_scales(MW, BLOCK) + m * 8 + 4, r.at1 + m * r.more);
            }
        }
        if (BLOCK) {
            ++r.at0;
            ++r.at1;
        }
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
// A stage's scales, once its copies and the warp have met.
template <bool BLOCK, int MW>
__device__ __forceinline__ void w8_read_scales(const W8Ring& r, int stage, float (&s0)[MW], float (&s1)[MW]) {
#pragma unroll
    for (int m = 0; m < MW; ++m) {
        if (BLOCK && m) {  // sixteen rows lie in one block of 128, and so do thirty-two
            s0[m] = s0[0];
            s1[m] = s1[0];
        } else {
            asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(s0[m]), "=f"(s1[m]) : "r"(r.scales + stage * w8_scales(MW, BLOCK) + m * 8) : "memory");
        }
    }
}

// What a lane reads beside the weights, an item (half an item, with two groups of columns) ahead: its columns at its K indices.  Where a block has no such row they are
// the first one's: nobody stores what comes of them, and nothing has to be filled with zeros.
template <int P, int RB>
using W8Columns = uint4[RB][P][4 / RB];
template <int P, int RB>
__device__ __forceinline__ void w8_copy_columns(W8Columns<P, RB>& to, const W8Columns<P, RB>& from) {
#pragma unroll
    for (int c = 0; c < RB; ++c)
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < 4 / RB; ++i) to[c][p][i] = from[c][p][i];
}
template <int P, int RB>
struct W8Ahead {
    const void* col[RB];
    int k;  // 128-element block

    // RAW: the column is f32, 32 of its values to b, for halves().  Else it is f16, `stride` elements between the parts.
    template <bool RAW>
    __device__ __forceinline__ void fetch(W8Columns<P, RB>& b, int stride, int half) const {
        if constexpr (RAW) {
            static_assert(P == 2 && RB == 1, "32 values of f32 are two parts of f16");
#pragma unroll
            for (int i = 0; i < 8; ++i)
                b[0][i >> 2][i & 3] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const float*>(col[0]) + k * 128 + (i >> 2) * 64 + (i & 3) * 4));
        } else {
#pragma unroll
            for (int c = 0; c < RB; ++c)
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                    for (int i = 0; i < 4 / RB; ++i)
                        b[c][p][i] = *reinterpret_cast<const uint4*>(static_cast<const __half*>(col[c]) + p * stride + k * 128 + (half + (i >> 1)) * 64 + (i & 1) * 8);
        }
    }
};

// 32 values of f32 as they were fetched, times `up`, as value and remainder.
__device__ __forceinline__ void w8_halves(uint4 (&b)[2][4], float up) {
    uint4 raw[2][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i >> 2][i & 3] = b[i >> 2][i & 3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // eight values: the i-th sixteen bytes of either part
        const uint4 &v = raw[i >> 1][2 * (i & 1)], &w = raw[i >> 1][2 * (i & 1) + 1];
        uint32_t out[4][2];
        w8_split<2>(__uint_as_float(v.x) * up, __uint_as_float(v.y) * up, out[0]);
        w8_split<2>(__uint_as_float(v.z) * up, __uint_as_float(v.w) * up, out[1]);
        w8_split<2>(__uint_as_float(w.x) * up, __uint_as_float(w.y) * up, out[2]);
        w8_split<2>(__uint_as_float(w.z) * up, __uint_as_float(w.w) * up, out[3]);
        b[0][i] = make_uint4(out[0][0], out[1][0], out[2][0], out[3][0]);
        b[1][i] = make_uint4(out[0][1], out[1][1], out[2][1], out[3][1]);
    }
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

// ------------------------------------------------------------------------------------------------ spans of whole tiles: gate_up; down, general form
// FEW: one CTA an SM, which brings x of bf16 to f16 itself.  RB: groups of eight rows that a block has at most.
template <typename T, bool BLOCK, bool SELF, bool DOWN, bool FEW, int MW, int RB>
__global__ void __launch_bounds__(kW8Threads, 2) moe_w8_tiles_kernel(const __grid_constant__ W8Params p) {
    constexpr int P = DOWN ? kW8PartsH : 1, kSums = MW * RB, kRing = w8_ring(MW, FEW), kDepth = w8_depth(MW, FEW), kStage = w8_stage(MW, FEW, BLOCK);
    constexpr bool OWN = FEW && !std::is_same<T, __half>::value;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float own_scale[kW8SelfTokens];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, j = lane & 3;
    float4* part = reinterpret_cast<float4*>(smem + kW8Warps * kRing);  // [warps][first, last tile][RB][MW][32]
    unsigned char* scales = reinterpret_cast<unsigned char*>(part + kW8Warps * 2 * kSums * 32);  // [warps][kDepth]
    W8Plan& plan = *reinterpret_cast<W8Plan*>(scales + kW8Warps * kStage);
    __half* own = reinterpret_cast<__half*>(reinterpret_cast<unsigned char*>(&plan) + (sizeof(W8Plan) + 15) / 16 * 16);  // [T][K + 8]

    if (!DOWN) {  // (the launches ahead of the down product each waited before they let the next start: the blocks may be read and weights asked for)
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // behind the wait: what follows may read this launch's inputs early
    }
    const int K = DOWN ? p.I : p.H, items = K / 128, own_stride = K + 8;
    if (SELF) {
        // the first four warps route, the others bring x to f16
        w8_picks(p, plan, OWN ? 4 : kW8Warps);
        if (OWN && warp >= 4)
            w8_rows_parts<1>(static_cast<const T*>(p.x), p.T, K, warp - 4, 4,
                             [&](int t, int, int i, uint2 four) { *reinterpret_cast<uint2*>(own + static_cast<size_t>(t) * own_stride + i) = four; },
                             [&](int t, float down) { own_scale[t] = down; });
        w8_group(p, plan);
    }
    const int n_blocks = SELF ? plan.n_blocks : *p.n_blocks;
    const int tiles = DOWN ? p.H / (16 * MW) : p.I / (8 * MW);  // of a block
    using Int = typename std::conditional<SELF, int, int64_t>::type;  // up to 512 blocks of 65536-wide experts: 32 bits, whose divisions are short
    const Int units = static_cast<Int>(n_blocks) * tiles;
    const Int u0 = units * static_cast<int>(blockIdx.x) / static_cast<int>(gridDim.x);
    const int span = static_cast<int>(units * static_cast<int>(blockIdx.x + 1) / static_cast<int>(gridDim.x) - u0);
    const Int total = static_cast<Int>(span) * items;
    auto share = [&](int w) { return total * w / kW8Warps; };
    const Int q0 = share(warp);
    const int n = static_cast<int>(share(warp + 1) - q0);
    const int first = static_cast<int>(q0 / items), skip = static_cast<int>(q0 - static_cast<Int>(first) * items);
    const int block0 = static_cast<int>(u0 / tiles), tile0 = static_cast<int>(u0 - static_cast<Int>(block0) * tiles);

    // tile `rel` of the span
    struct Tile {
        int block, chan;
    };
    auto tile_of = [&](int rel) {
        const int over = (tile0 + rel) / tiles;
        return Tile{block0 + over, tile0 + rel - over * tiles};
    };
    W8Ring ring;
    ring.base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * kRing + lane * 16;
    ring.step = (DOWN ? 16 : 8) * K;
    ring.scales = static_cast<uint32_t>(__cvta_generic_to_shared(scales)) + warp * kStage + g * (w8_scales(MW, BLOCK) / 8);
    ring.more = DOWN ? 16 : 8;
    ring.left = n;
    ring.room = items - skip;
    int ask = first;  // tile of the next item to ask for
    auto rows_of = [&](int k) {
        const Tile t = tile_of(ask);
        const int expert = w8_block<SELF>(p, plan, t.block).expert, rows = DOWN ? p.H : 2 * p.I, r0 = t.chan * MW * (DOWN ? 16 : 8) + g;
        ring.top = p.w + (static_cast<size_t>(expert) * rows + r0) * K + k * 128 + 16 * j;
        ring.bottom = ring.top + static_cast<size_t>(DOWN ? 8 : p.I) * K;
        if (BLOCK) {
            ring.at0 = p.scale + (static_cast<size_t>(expert) * (rows / 128) + (DOWN ? t.chan * MW / 8 : t.chan * MW / 16)) * items + k;
            ring.at1 = DOWN ? ring.at0 : ring.at0 + static_cast<size_t>(p.I / 128) * items;
        } else {
            ring.at0 = p.scale + static_cast<size_t>(expert) * rows + r0;
            ring.at1 = ring.at0 + (DOWN ? 8 : p.I);
        }
    };
    auto open = [&]() {
        ++ask;
        rows_of(0);
    };
    if (n > 0) rows_of(skip);
#pragma unroll 1
    for (int d = 0; d < kDepth; ++d) w8_issue<BLOCK, MW>(ring, d, items, open);

    if (DOWN) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    W8Ahead<P, RB> next;
    W8Columns<P, RB> b0, b1;  // the next ones, and those in hand (the second half's)
    int at = first;  // the tile that `next` is of
    next.k = skip;
    auto enter = [&]() {
        const Tile t = tile_of(at);
        const W8Block blk = w8_block<SELF>(p, plan, t.block);
#pragma unroll
        for (int c = 0; c < RB; ++c) {
            const int row = blk.row0 + (g + 8 * c < blk.count ? g + 8 * c : 0);
            if (DOWN) {
                next.col[c] = p.h16 + static_cast<size_t>(row) * P * K + 16 * j;
            } else {
                const int token = SELF ? plan.token[row] : p.rows[row] / p.topk;
                next.col[c] = (OWN ? own + static_cast<size_t>(token) * own_stride : p.x16 + static_cast<size_t>(token) * K) + 16 * j;
            }
        }
    };
    auto fetch = [&](W8Columns<P, RB>& b, int half) { next.template fetch<false>(b, K, half); };
    // the finished sums of a tile (lane: channels g and g + 8, or gate and up of channel g; rows 2 j, 2 j + 1)
    auto finish = [&](int rel, const float (&sum)[RB][MW][4]) {
        const Tile t = tile_of(rel);
        const W8Block blk = w8_block<SELF>(p, plan, t.block);
#pragma unroll
        for (int ci = 0; ci < 2 * RB; ++ci) {
            const int c = ci >> 1, i = ci & 1, r = 8 * c + 2 * j + i;
            const bool in = r < blk.count;
            if (DOWN) {
                if (!in) continue;
                const float down = __ldcg(p.h_scale + blk.row0 + r);
                float* to = p.rows_out + static_cast<size_t>(p.rows[blk.row0 + r]) * p.H + t.chan * 16 * MW + g;
#pragma unroll
                for (int m = 0; m < MW; ++m) {
                    to[16 * m] = sum[c][m][i] * down;
                    to[16 * m + 8] = sum[c][m][2 + i] * down;
                }
            } else {
                float big = 0.f;
                if (in) {
                    const int token = SELF ? plan.token[blk.row0 + r] : p.rows[blk.row0 + r] / p.topk;
                    const float down = OWN ? own_scale[token] : p.x_scale ? __ldcg(p.x_scale + token) : 1.f;
#pragma unroll
                    for (int m = 0; m < MW; ++m) {
                        const float gate = sum[c][m][i] * down, up_ = sum[c][m][2 + i] * down, h = gate / (1.f + expf(-gate)) * up_;
                        p.h[static_cast<size_t>(blk.row0 + r) * p.I + (t.chan * MW + m) * 8 + g] = h;
                        big = fabsf(h) < INFINITY ? fmaxf(big, fabsf(h)) : big;
                    }
                }
                if (p.h_max) {  // the maximum does not depend on the order of its atomics
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, off));
                    if (in && g == 0) atomicMax(p.h_max + blk.row0 + r, __float_as_uint(big));
                }
            }
        }
    };

    if (n > 0) {
        enter();
        fetch(b0, 0);
    }
    int stage = 0;
    int rel = first, it = skip;
    for (int i = 0; i < n;) {
        const int stretch = min(items - it, n - i);
        float sum[RB][MW][4] = {};
        for (int c = 0; c < stretch; ++c) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
            __syncwarp();
            float s0[MW], s1[MW];
            w8_read_scales<BLOCK, MW>(ring, stage, s0, s1);
            const uint32_t slot = ring.base + stage * MW * 2048;
            auto advance = [&](W8Columns<P, RB>& to) {
                if (i + c + 1 < n) {
                    if (++next.k == items) {
                        next.k = 0;
                        ++at;
                        enter();
                    }
                    fetch(to, 0);
                }
            };
            if constexpr (RB == 2) {  // the halves of an item
                fetch(b1, 1);
                w8_item<P, MW, RB>(slot, b0, s0, s1, sum);
                advance(b0);
                w8_item<P, MW, RB>(slot + 1024, b1, s0, s1, sum);
            } else {
                w8_copy_columns<P, RB>(b1, b0);
                advance(b0);
                w8_item<P, MW, RB>(slot, b1, s0, s1, sum);
            }
            __syncwarp();
            w8_issue<BLOCK, MW>(ring, stage, items, open);
            stage = stage + 1 == kDepth ? 0 : stage + 1;
        }
        if (stretch == items) {
            finish(rel, sum);
        } else {  // another warp has a part of the tile
#pragma unroll
            for (int q = 0; q < kSums; ++q) {
                const float(&v)[4] = sum[q / MW][q % MW];
                part[((warp * 2 + (rel == first ? 0 : 1)) * kSums + q) * 32 + lane] = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
        i += stretch;
        it = 0;
        ++rel;
    }
    __syncthreads();
    // the shared tiles, in the order of the warps that have a part
    for (int t = warp; t < span; t += kW8Warps) {
        const Int lo_item = static_cast<Int>(t) * items, hi_item = lo_item + items;
        float sum[RB][MW][4] = {};
        int parts = 0;
        for (int w = 0; w < kW8Warps; ++w) {
            const Int a = share(w), b = share(w + 1);
            if (a >= hi_item || b <= lo_item || a == b || (a <= lo_item && b >= hi_item)) continue;
            ++parts;
#pragma unroll
            for (int q = 0; q < kSums; ++q) {
                const float4 v = part[((w * 2 + (a >= lo_item ? 0 : 1)) * kSums + q) * 32 + lane];
                float(&to)[4] = sum[q / MW][q % MW];
                to[0] += v.x;
                to[1] += v.y;
                to[2] += v.z;
                to[3] += v.w;
            }
        }
        if (parts) finish(t, sum);
    }
}

// ------------------------------------------------------------------------------------------------ down, sixteen channels of all blocks
__device__ __forceinline__ float w8_peer(const float* mine, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

template <typename T, bool BLOCK, bool OWN, int MW>
__global__ void __launch_bounds__(kW8Threads, 2) moe_w8_down_kernel(const __grid_constant__ W8Params p) {
    constexpr bool kRaw = !OWN;
    constexpr int P = kW8PartsH, kRing = w8_ring(MW, OWN), kDepth = w8_depth(MW, OWN), kStage = w8_stage(MW, OWN, BLOCK), kChan = 16 * MW;
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, j = lane & 3;
    float* sums = reinterpret_cast<float*>(smem + kW8Warps * kRing);  // [warps][T][kChan]
    unsigned char* scales = reinterpret_cast<unsigned char*>(sums + kW8Warps * p.T * kChan);  // [warps][kDepth]
    W8Plan& plan = *reinterpret_cast<W8Plan*>(scales + kW8Warps * kStage);
    __half* own = reinterpret_cast<__half*>(reinterpret_cast<unsigned char*>(&plan) + (sizeof(W8Plan) + 15) / 16 * 16);  // [picks][P][I + 8]
    uint32_t rank, ctas;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    // The launches before this one each waited for what came before them ahead of letting the next start, so the logits may be read here and the
    // weights asked for; what they compute is read behind the wait.
    w8_picks(p, plan, kW8Warps);
    w8_group(p, plan);
    for (int i = tid; i < kW8Warps * p.T * kChan; i += kW8Threads) sums[i] = 0.f;
    __syncthreads();
    const int items = p.I / 128, chan = static_cast<int>(blockIdx.x / ctas) * kChan, own_stride = p.I + 8;
    const int total = plan.n_blocks * items, shares = kW8Warps * ctas, mine = rank * kW8Warps + warp;
    const int q0 = total * mine / shares, n = total * (mine + 1) / shares - q0;  // (512 blocks of 512 items, 64 shares at most)
    const int first = q0 / items, skip = q0 - first * items;
    W8Ring ring;
    ring.base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * kRing + lane * 16;
    ring.step = 16 * p.I;
    ring.scales = static_cast<uint32_t>(__cvta_generic_to_shared(scales)) + warp * kStage + g * (w8_scales(MW, BLOCK) / 8);
    ring.more = 16;
    ring.left = n;
    ring.room = items - skip;
    int ask = first;
    auto rows_of = [&](int b, int k) {
        ring.top = p.w + (static_cast<size_t>(plan.expert[b]) * p.H + chan + g) * p.I + k * 128 + 16 * j;
        ring.bottom = ring.top + static_cast<size_t>(8) * p.I;
        if (BLOCK) {
            ring.at0 = ring.at1 = p.scale + (static_cast<size_t>(plan.expert[b]) * (p.H / 128) + chan / 128) * items + k;
        } else {
            ring.at0 = p.scale + static_cast<size_t>(plan.expert[b]) * p.H + chan + g;
            ring.at1 = ring.at0 + 8;
        }
    };
    if (n > 0) rows_of(ask, skip);
    auto open = [&]() { rows_of(++ask, 0); };
#pragma unroll 1
    for (int d = 0; d < kDepth; ++d) w8_issue<BLOCK, MW>(ring, d, items, open);

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (OWN) {
        // (a row's factor goes to its weight in the token's sum)
        const int picks = plan.row0[plan.n_blocks - 1] + plan.count[plan.n_blocks - 1];
        w8_rows_parts<P>(p.h, picks, p.I, warp, kW8Warps,
                         [&](int r, int q, int i, uint2 four) { *reinterpret_cast<uint2*>(own + (static_cast<size_t>(r) * P + q) * own_stride + i) = four; },
                         [&](int r, float down) { plan.score[r] *= down; });
        __syncthreads();
    }
    W8Ahead<P, 1> next;
    W8Columns<P, 1> b0, b1;  // the next ones, and those in hand
    int at = first;
    next.k = skip;
    float up = 1.f;  // what brings this lane's row of h to f16
    auto enter = [&]() {
        const int row0 = plan.row0[at];
        const int row = row0 + (g < plan.count[at] ? g : 0);
        if (OWN) {
            next.col[0] = own + static_cast<size_t>(row) * P * own_stride + 16 * j;
        } else {
            next.col[0] = p.h + static_cast<size_t>(row) * p.I + 16 * j;
            up = w8_up(__uint_as_float(__ldcg(p.h_max + row)));
        }
    };
    auto fetch = [&](W8Columns<P, 1>& b) { next.template fetch<kRaw>(b, own_stride, 0); };
    if (n > 0) {
        enter();
        fetch(b0);
    }
    float* my_sums = sums + warp * p.T * kChan;
    int stage = 0;
    int rel = first, it = skip;
    for (int i = 0; i < n;) {
        const int stretch = min(items - it, n - i);
        const int row0 = plan.row0[rel], count = plan.count[rel];
        float down[2] = {1.f, 1.f};
        if (!OWN) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (2 * j + e < count) down[e] = 1.f / w8_up(__uint_as_float(__ldcg(p.h_max + row0 + 2 * j + e)));
        }
        float sum[1][MW][4] = {};
        for (int c = 0; c < stretch; ++c) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
            __syncwarp();
            float s0[MW], s1[MW];
            w8_read_scales<BLOCK, MW>(ring, stage, s0, s1);
            w8_copy_columns<P, 1>(b1, b0);
            const float now_up = up;
            if (i + c + 1 < n) {
                if (++next.k == items) {
                    next.k = 0;
                    ++at;
                    enter();
                }
                fetch(b0);
            }
            if constexpr (kRaw) w8_halves(b1[0], now_up);
            w8_item<P, MW, 1>(ring.base + stage * MW * 2048, b1, s0, s1, sum);
            __syncwarp();
            w8_issue<BLOCK, MW>(ring, stage, items, open);
            stage = stage + 1 == kDepth ? 0 : stage + 1;
        }
        // this warp's part of the block's rows, weighted, to its tokens' sums (the rows of a block are different tokens)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 2 * j + e;
            if (r < count) {
                const float weight = plan.score[row0 + r] * down[e];
                float* to = my_sums + plan.token[row0 + r] * kChan + g;
#pragma unroll
                for (int m = 0; m < MW; ++m) {
                    to[16 * m] += weight * sum[0][m][e];
                    to[16 * m + 8] += weight * sum[0][m][2 + e];
                }
            }
        }
        __syncwarp();
        i += stretch;
        it = 0;
        ++rel;
    }
    __syncthreads();
    // the warps' sums in warp order, the CTAs' in rank order
    for (int i = tid; i < p.T * kChan; i += kW8Threads) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kW8Warps; ++w) v += sums[w * p.T * kChan + i];
        sums[i] = v;
    }
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
    for (int i = rank * kW8Threads + tid; i < p.T * kChan; i += ctas * kW8Threads) {
        float v = 0.f;
        for (uint32_t c = 0; c < ctas; ++c) v += ctas > 1 ? w8_peer(sums + i, c) : sums[i];
        static_cast<T*>(p.y)[static_cast<size_t>(i / kChan) * p.H + chan + i % kChan] = from_float<T>(v);
    }
    if (ctas > 1) {  // no CTA leaves while another may read its sums
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

// y[t] = sum_j score[t, j] rows[t topk + j], four channels a thread, picks in the order of their logits.
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
    __half *x16, *h16;
    float *x_scale, *h, *shares, *rows_out, *h_scale;
    uint32_t* h_max;
    int32_t *ids, *rows, *n_blocks;
    GroupBlock* blocks;
    size_t bytes;
};

// (wider experts than 65536: the general form, whose indices have 64 bits)
static bool w8_self(int64_t T, int64_t E, int64_t H, int64_t I) { return T <= kW8SelfTokens && E <= kW8SelfExperts && H <= 65536 && I <= 65536; }

static W8Workspace w8_carve(void* base, int64_t T, int64_t E, int64_t topk, int64_t H, int64_t I) {
    W8Workspace w = {};
    unsigned char* b = static_cast<unsigned char*>(base);
    size_t o = 0;
    auto take = [&](size_t bytes) {
        void* at = b + o;
        o += w8_align(bytes);
        return at;
    };
    const size_t R = static_cast<size_t>(T) * topk;
    w.h = static_cast<float*>(take(R * I * 4));
    w.h_max = static_cast<uint32_t*>(take(R * 4));
    w.x16 = static_cast<__half*>(take(static_cast<size_t>(T) * H * 2));
    w.x_scale = static_cast<float*>(take(static_cast<size_t>(T) * 4));
    w.ids = static_cast<int32_t*>(take(R * 4));
    w.shares = static_cast<float*>(take(R * 4));
    if (!w8_self(T, E, H, I)) {
        w.rows = static_cast<int32_t*>(take(R * 4));
        w.n_blocks = static_cast<int32_t*>(take(4));
        w.blocks = static_cast<GroupBlock*>(take(static_cast<size_t>(group_max_blocks(static_cast<int64_t>(R), E, kW8BlockRows, false)) * sizeof(GroupBlock)));
        w.rows_out = static_cast<float*>(take(R * H * 4));
        w.h16 = static_cast<__half*>(take(R * kW8PartsH * I * 2));
        w.h_scale = static_cast<float*>(take(R * 4));
    }
    w.bytes = o;
    return w;
}

template <typename... P, typename... A>
static int w8_launch(void (*kernel)(P...), int64_t grid, int cluster, size_t smem, cudaStream_t stream, A... args) {
    if (smem > kSmemUnasked) EQ_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kW8Threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    EQ_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
    return EQ_OK;
}

// Which kernels a call takes.
struct W8Form {
    bool self;  // the CTAs group the picks, two products and nothing else
    bool own;   // and route and bring x and silu * up to f16 as well
    bool wide;  // thirty-two rows a warp
    int rb;     // groups of eight rows of a block, general form
};
constexpr size_t kW8Plan = (sizeof(W8Plan) + 15) / 16 * 16;
// Dynamic shared memory of a CTA; with few the activations come on top.
static size_t w8_tiles_smem(int mw, int rb, bool few, bool block) { return static_cast<size_t>(kW8Warps) * (w8_ring(mw, few) + w8_stage(mw, few, block) + 2 * mw * rb * 32 * sizeof(float4)); }
static size_t w8_down_smem(int64_t T, int mw, bool few, bool block) {
    return static_cast<size_t>(kW8Warps) * (w8_ring(mw, few) + w8_stage(mw, few, block) + static_cast<size_t>(T) * 16 * mw * sizeof(float)) + kW8Plan;
}
static size_t w8_own_x(int64_t T, int64_t H, bool f16) { return f16 ? 0 : static_cast<size_t>(T) * (H + 8) * 2; }
static size_t w8_own_h(int64_t R, int64_t I) { return static_cast<size_t>(R) * kW8PartsH * (I + 8) * 2; }

static W8Form w8_form(int64_t T, int64_t E, int64_t topk, int64_t H, int64_t I, bool f16) {
    W8Form f;
    const int64_t R = T * topk, sms = sm_count();
    f.self = w8_self(T, E, H, I);
    // Thirty-two rows a warp where there are enough of them: half as many reads of the activations, which lie in L1 and L2, for the same weights.  us a layer with
    // sixteen and thirty-two, by R I / 16.  H from 1280 on: 16 experts of 2048 x 2816, top 4, 1408 40.1 : 36.6, 5632 67 : 62, 22528 110 : 93; 128 of 2048 x 768,
    // top 8, 768 28.4 : 27.5, 2304 55 : 50, 12288 135 : 119; 128 of 1280 x 768, 768 24.6 : 23.2, 2304 47 : 41; below, nothing in it (32 of 2048 x 512, top 4, 384
    // 18.9 : 18.9; 8 of 2048 x 256, top 2, 256 14.6 : 15.7).  Narrower layers have few slabs of thirty-two channels, in clusters of eight: 32 of 1024 x 512, 384
    // 16.0 : 20.7, 768 18.6 : 24.1, 1536 23.2 : 23.4; 128 of 1024 x 768, 2304 35.5 : 32.9, 7680 68 : 59, 12288 (32 tokens) 80 : 90; of 640 x 768, 4608 43 : 38.
    // And clusters of four do not pack into all slots of two CTAs an SM: 256 experts of 2304 x 896, top 8, whose down product has 288, 1344 42.8 : 47.1, 2688
    // 71.7 : 76.9, 14336 225 : 260 (with 272, of 2176 x 896, 42.1 : 39.1, 69.9 : 62.8; 209 : 237 at 32 tokens).
    const int64_t fours = 4 * (H / 32);
    f.wide = R * (I / 16) >= (H >= 1280 ? 4 : 16) * sms && !(fours <= 2 * sms && fours > 2 * sms * 15 / 16);
    // CTAs that route and convert for themselves, no launch ahead of them: where one of either product, with its activations, fits an SM beside the other
    // (228 KB; 1 KB of each is the system's, 192 bytes of both are static), and the down product's slabs of sixteen channels are no more than SMs.  Without
    // and with, us: 128 experts of 2048 x 768, a token, top 8 18.7 : 17.7, two, top 4 20.7 : 18.9; 64 of 2048 x 1024, three of f16, top 2 19.4 : 16.4, four (too large
    // by 1 KB) 22.3 : 23.4; 8 of 2048 x 2048, two of f16 19.8 : 17.3; 8 of 2304 x 512, top 8, two of f16 (96 bytes are left) 18.4 : 16.9; 32 of 1024 x 512, top 4,
    // three 15.9 : 15.7, four (too large) 16.4 : 18.4; more slabs than SMs: 8 of 4096 x 4096, one, top 1 20.9 : 22.8, 32 of 5120 x 768, one of f16, top 8 32.3 : 45.3.
    constexpr size_t kSm = 228 * 1024, kBeside = 2 * 1024 + 256;
    f.own = f.self && !f.wide && H / 16 <= sms &&
            w8_tiles_smem(1, 1, true, true) + kW8Plan + w8_own_x(T, H, f16) + w8_down_smem(T, 1, true, true) + w8_own_h(R, I) + kBeside <= kSm;
    // Sixteen rows a block where experts have that many: the weights of an expert with nine to sixteen rows are read and expanded once and not twice, but half as
    // far ahead.  128 experts of 2048 x 768, top 8, us a layer with 8 and 16: 96 tokens 149 and 171, 128 174 and 176, 144 180 and 180, 160 193 and 180, 200 236 and
    // 189, 256 298 and 230; 64 experts, top 6: 96 tokens 161 and 165, 128 193 and 182.
    f.rb = R > 9 * E ? 2 : 1;
    return f;
}

template <typename T, bool BLOCK>
static int w8_forward(W8Params p, const uint8_t* gate_up, const float* gate_up_scale, const uint8_t* down, const float* down_scale, const W8Workspace& w,
                      cudaStream_t stream) {
    const size_t plan = kW8Plan;
    const int64_t R = static_cast<int64_t>(p.T) * p.topk;
    constexpr bool f16 = std::is_same<T, __half>::value;  // x is read as it is
    const W8Form form = w8_form(p.T, p.E, p.topk, p.H, p.I, f16);
    const bool self = form.self, wide = form.wide, own = form.own;
    const int rb = form.rb;
    const size_t own_x = w8_own_x(p.T, p.H, f16), own_h = w8_own_h(R, p.I);
    const int64_t sms = sm_count(), most = 2 * sms;
    int st = EQ_OK;
    p.h_max = self && !own ? w.h_max : nullptr;
    p.h16 = w.h16;
    p.h_scale = w.h_scale;
    if (own) {
        p.x16 = static_cast<const __half*>(p.x);  // of f16
    } else {
        auto prep = [&](auto kernel) { return w8_launch(kernel, p.T, 1, 0, stream, p, w.ids, w.shares, w.x16, w.x_scale); };
        st = p.E <= 128 ? prep(w8_prep_kernel<T, 4>) : p.E <= 256 ? prep(w8_prep_kernel<T, 8>) : prep(w8_prep_kernel<T, 32>);
        p.ids = w.ids;
        p.shares = w.shares;
        p.x16 = f16 ? static_cast<const __half*>(p.x) : w.x16;
        p.x_scale = f16 ? nullptr : w.x_scale;
        if (st == EQ_OK && !self) st = group_rows_launch(w.ids, static_cast<int>(R), p.E, false, rb * kW8BlockRows, false, w.blocks, w.n_blocks, w.rows, nullptr, stream);
    }
    if (st != EQ_OK) return st;
    p.w = gate_up;
    p.scale = gate_up_scale;
    auto smem = [](int mw, int rb = 1, bool few = false) { return w8_tiles_smem(mw, rb, few, BLOCK); };
    if (self) {
        const int64_t tiles = R * (p.I / (wide ? 16 : 8)), at_once = own ? sms : most, grid = tiles < at_once ? tiles : at_once;
        if (own) st = w8_launch(moe_w8_tiles_kernel<T, BLOCK, true, false, true, 1, 1>, grid, 1, smem(1, 1, true) + plan + own_x, stream, p);
        else if (wide) st = w8_launch(moe_w8_tiles_kernel<T, BLOCK, true, false, false, 2, 1>, grid, 1, smem(2) + plan, stream, p);
        else st = w8_launch(moe_w8_tiles_kernel<T, BLOCK, true, false, false, 1, 1>, grid, 1, smem(1) + plan, stream, p);
    } else {
        st = rb == 2 ? w8_launch(moe_w8_tiles_kernel<T, BLOCK, false, false, false, 2, 2>, most, 1, smem(2, 2), stream, p)
                     : w8_launch(moe_w8_tiles_kernel<T, BLOCK, false, false, false, 2, 1>, most, 1, smem(2), stream, p);
    }
    if (st != EQ_OK) return st;
    p.w = down;
    p.scale = down_scale;
    if (self) {
        const int mw = wide ? 2 : 1;
        const int64_t slabs = p.H / (16 * mw);
        int cluster = 8;  // two CTAs an SM at most, one beside the launch ahead
        while (cluster > 1 && slabs * cluster > (own ? sms : most)) cluster /= 2;
        const size_t bytes = w8_down_smem(p.T, mw, own, BLOCK);
        if (wide) return w8_launch(moe_w8_down_kernel<T, BLOCK, false, 2>, slabs * cluster, cluster, bytes, stream, p);
        return own ? w8_launch(moe_w8_down_kernel<T, BLOCK, true, 1>, slabs * cluster, cluster, bytes + own_h, stream, p)
                     : w8_launch(moe_w8_down_kernel<T, BLOCK, false, 1>, slabs * cluster, cluster, bytes, stream, p);
    }
    st = w8_launch(w8_parts_kernel, R, 1, 0, stream, static_cast<const float*>(w.h), p.I, w.h16, w.h_scale);
    if (st != EQ_OK) return st;
    st = rb == 2 ? w8_launch(moe_w8_tiles_kernel<T, BLOCK, false, true, false, 2, 2>, most, 1, smem(2, 2), stream, p)
                 : w8_launch(moe_w8_tiles_kernel<T, BLOCK, false, true, false, 2, 1>, most, 1, smem(2), stream, p);
    if (st != EQ_OK) return st;
    const int64_t vecs = static_cast<int64_t>(p.T) * p.H / 4;
    return w8_launch(moe_w8_combine_kernel<T>, ceil_div(vecs, 256), 1, 0, stream, reinterpret_cast<const float4*>(w.rows_out), static_cast<const float*>(w.shares), vecs, p.H / 4,
                     p.topk, static_cast<T*>(p.y));
}

}  // namespace eq

using namespace eq;

extern "C" size_t eq_moe_w8a16_workspace_bytes(int64_t T, int64_t E, int64_t topk, int64_t H, int64_t I) {
    if (T <= 0 || E <= 0 || topk <= 0 || H <= 0 || I <= 0) return 0;
    return w8_carve(nullptr, T, E, topk, H, I).bytes;
}

extern "C" const char* eq_moe_w8a16_kernel(int64_t T, int64_t E, int64_t topk, int64_t H, int64_t I, int act_dtype) {
    const W8Form f = w8_form(T, E, topk, H, I, act_dtype == EQ_F16);
    if (f.self) return f.own ? "moe_w8_down_kernel, own" : f.wide ? "moe_w8_down_kernel, wide" : "moe_w8_down_kernel";
    return f.rb == 2 ? "moe_w8_tiles_kernel, sixteen rows" : "moe_w8_tiles_kernel, eight rows";
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
    p.h = w.h;
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
