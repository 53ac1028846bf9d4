// The router of a mixture of experts: the `top` largest of each token's scores, their weights, and all (token, expert) pairs sorted by expert for the experts' products.
//
// A wavefront holds the logits of a token in registers, one to sixteen a lane, and takes the largest `top` times: a key (the value's bits in an order that integers compare right, above
// the index inverted, so that equal scores go by rising index) is reduced over the lanes by DPP steps.  softmax and sigmoid rise with the logit, so the logits themselves decide; with a bias on the
// scores the choice is made in 64 bits, where no two scores that differ round to one.
//
// The sort is stable and counts: every workgroup counts its pairs by expert; what lies before a pair is the pairs of lower experts, those of its expert in workgroups and wavefronts before, and those in
// lower lanes of its own, found by comparing the bits of the expert's number over the lanes.  No atomics decide a place, so two calls give the same order.  A few tokens, or 1024 pairs whose experts
// are given, one launch does both; more take a second one for the places.
//
// What bounds it: latency (one token: the way in, `top` reductions of some forty instructions one after the other, the way out).  In a trace, one fp32 token, 8 of 64 experts 3.6 us; 4099 bf16 tokens, 8 of
// 128 8.5 us (vector units busy 0.64) and 7.5 for the places, 15.5 for both as called.
#include <algorithm>

#include "experts.h"

namespace qmm {

namespace {

constexpr int kRouteThreads = 1024, kRouteWaves = kRouteThreads / 64;
constexpr int kRouteBlocks = 512;  // workgroups at most: each adds up the counts of those before it

template <int CTRL>
__device__ __forceinline__ uint64_t dpp_move64(uint64_t v) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, 0xf, 0xf, true) << 32 | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ float lane32(float v, int lane) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane)); }
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
    v = larger(v, dpp_move64<0xB1>(v));
    v = larger(v, dpp_move64<0x4E>(v));
    v = larger(v, dpp_move64<0x141>(v));
    v = larger(v, dpp_move64<0x140>(v));
    return larger(larger(lane64(v, 0), lane64(v, 16)), larger(lane64(v, 32), lane64(v, 48)));
}

// Numbers in the order of the values; -0 is 0, NaN below everything, never 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 1u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_of(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return x != x ? 1ull : (b >> 63) ? ~b : b | 1ull << 63;
}

struct RouteCall {
    int64_t stride;
    int tokens, experts, top;
    bool sigmoid, renormalize;
    float scale;
    const float* bias;
};

// One token by one wavefront; lane j holds expert 64 i + j in x[i].  Its j-th expert, in lane j.
template <int VPL, typename T>
__device__ __forceinline__ int route_token(const T* __restrict__ logits, const RouteCall& c, int64_t token, int lane, int32_t* __restrict__ ids, float* __restrict__ weights) {
    float x[VPL];
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const int e = 64 * i + lane;
        x[i] = load_f32(logits, token * c.stride + min(e, c.experts - 1));  // (all loads at once)
    }
#pragma unroll
    for (int i = 0; i < VPL; i++) x[i] = 64 * i + lane < c.experts ? x[i] : -__builtin_inff();
    float m = x[0];
#pragma unroll
    for (int i = 1; i < VPL; i++) m = fmaxf(m, x[i]);
    m = fmaxf(m, dpp_move<0xB1>(m));
    m = fmaxf(m, dpp_move<0x4E>(m));
    m = fmaxf(m, dpp_move<0x141>(m));
    m = fmaxf(m, dpp_move<0x140>(m));
    m = fmaxf(fmaxf(lane32(m, 0), lane32(m, 16)), fmaxf(lane32(m, 32), lane32(m, 48)));
    float chosen = 0.0f;  // lane j: the logit of the j-th choice
    int expert = -1;
    if (!c.bias) {
        uint64_t key[VPL];
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int e = 64 * i + lane;
            key[i] = e < c.experts ? (uint64_t)order_of(x[i]) << 32 | (uint32_t)~e : 0;
        }
        for (int j = 0; j < c.top; j++) {
            uint64_t best = key[0];
#pragma unroll
            for (int i = 1; i < VPL; i++) best = larger(best, key[i]);
            best = wave_max64(best);
#pragma unroll
            for (int i = 0; i < VPL; i++) key[i] = key[i] == best ? 0 : key[i];
            if (lane == j) {
                const uint32_t o = (uint32_t)(best >> 32);
                chosen = __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
                expert = (int)~(uint32_t)best;
            }
        }
    } else {
        double sum = 0.0;
        if (!c.sigmoid) {
#pragma unroll
            for (int i = 0; i < VPL; i++) sum += 64 * i + lane < c.experts ? exp((double)x[i] - (double)m) : 0.0;
#pragma unroll
            for (int mask = 32; mask; mask >>= 1) sum += __shfl_xor(sum, mask);
        }
        uint64_t key[VPL];
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int e = 64 * i + lane;
            if (e < c.experts) {
                const double score = c.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : exp((double)x[i] - (double)m) / sum;
                key[i] = order_of(score + (double)c.bias[e]);
            } else {
                key[i] = 0;
            }
        }
        for (int j = 0; j < c.top; j++) {
            uint64_t best = key[0];
#pragma unroll
            for (int i = 1; i < VPL; i++) best = larger(best, key[i]);
            best = wave_max64(best);
            // the lowest expert that has it
            int at = 0;
            float value = 0.0f;
            bool found = false;
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                const uint64_t has = __ballot(key[i] == best);
                if (!found && has) {
                    found = true;
                    const int owner = __builtin_ctzll(has);
                    at = 64 * i + owner;
                    value = __shfl(x[i], owner);
                    if (lane == owner) key[i] = 0;
                }
            }
            if (lane == j) chosen = value, expert = at;
        }
    }
    float w = 0.0f;
    if (lane < c.top) w = c.sigmoid ? 1.0f / (1.0f + expf(-chosen)) : chosen == -__builtin_inff() ? 0.0f : expf(chosen - m);  // (a NaN stays one)
    if (c.renormalize) {
        const float sum = wave_sum_dpp(w);
        w = sum == 0.0f ? 0.0f : w / sum;
    } else if (!c.sigmoid && m != -__builtin_inff()) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < VPL; i++) sum += 64 * i + lane < c.experts ? expf(x[i] - m) : 0.0f;
        w /= wave_sum_dpp(sum);
    }
    if (lane < c.top) {
        ids[token * c.top + lane] = expert;
        weights[token * c.top + lane] = w * c.scale;
    }
    return expert;
}

// LDS of the sort: counts[wavefronts][experts + 1], then start[experts + 1]
__device__ __forceinline__ int run_of(int id, int experts) { return id >= 0 && id < experts ? id : experts; }

// start: exclusive sums of start[0 .. count), by the first wavefront
__device__ __forceinline__ void exclusive_sums(int* start, int count, int wave, int lane) {
    __syncthreads();
    if (wave == 0) {
        const int per = (count + 63) / 64, from = min(lane * per, count), to = min(from + per, count);
        int mine = 0;
        for (int e = from; e < to; e++) mine += start[e];
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        sum -= mine;
        for (int e = from; e < to; e++) {
            const int v = start[e];
            start[e] = sum;
            sum += v;
        }
    }
    __syncthreads();
}

// Pairs from .. to - 1 to their places; start[e]: the place of the first of them with expert e.
__device__ __forceinline__ void place_pairs(const int32_t* __restrict__ ids, int next, int from, int to, int experts, int* counts, int* start, int32_t* __restrict__ order, int wave, int lane) {
    const int runs = experts + 1;
    int bits = 0;
    while ((1 << bits) < runs) bits++;
    for (int p0 = from; p0 < to; p0 += kRouteThreads) {
        for (int i = threadIdx.x; i < kRouteWaves * runs; i += kRouteThreads) counts[i] = 0;
        __syncthreads();
        const int p = p0 + (int)threadIdx.x;
        const bool here = p < to;
        const int run = here ? run_of(next, experts) : 0;
        uint64_t same = __ballot(here);
        for (int b = 0; b < bits; b++) {
            const uint64_t set = __ballot((run >> b) & 1);
            same &= (run >> b) & 1 ? set : ~set;
        }
        const int before = (int)__popcll(same & ((1ull << lane) - 1));
        if (here && before == 0) counts[wave * runs + run] = (int)__popcll(same);
        __syncthreads();
        if (here) {
            int place = start[run] + before;
            for (int w = 0; w < wave; w++) place += counts[w * runs + run];
            order[place] = p;
        }
        if (p0 + kRouteThreads < to) {
            next = ids[min(p + kRouteThreads, to - 1)];
            __syncthreads();
            for (int e = threadIdx.x; e < runs; e += kRouteThreads) {
                int sum = 0;
                for (int w = 0; w < kRouteWaves; w++) sum += counts[w * runs + e];
                start[e] += sum;
            }
            __syncthreads();
        }
    }
}

// Counts of this workgroup's pairs by expert into start (LDS).
__device__ __forceinline__ void count_pairs(const int32_t* __restrict__ ids, int from, int to, int experts, int* start) {
    for (int e = threadIdx.x; e <= experts; e += kRouteThreads) start[e] = 0;
    __syncthreads();
    for (int p = from + (int)threadIdx.x; p < to; p += kRouteThreads) atomicAdd(start + run_of(ids[p], experts), 1);
    __syncthreads();
}

// Counts of a workgroup in the workspace: rows of whole 16 bytes.
__host__ __device__ constexpr int counts_stride(int experts) { return (experts + 4) / 4 * 4; }

// The only workgroup: everything; one of several: its counts to its row of blocks.
__device__ __forceinline__ void count_or_place(const int32_t* ids, int from, int to, int experts, int* lds, int32_t* offsets, int32_t* order, int32_t* blocks, int wave, int lane) {
    int* const start = lds + kRouteWaves * (experts + 1);
    count_pairs(ids, from, to, experts, start);
    if (blocks) {
        for (int e = threadIdx.x; e <= experts; e += kRouteThreads) blocks[(int64_t)blockIdx.x * counts_stride(experts) + e] = start[e];
        return;
    }
    exclusive_sums(start, experts + 1, wave, lane);
    for (int e = threadIdx.x; e <= experts; e += kRouteThreads) offsets[e] = start[e];
    __syncthreads();
    place_pairs(ids, ids[min(from + (int)threadIdx.x, to - 1)], from, to, experts, lds, start, order, wave, lane);
}

template <int VPL, typename T>
__global__ __launch_bounds__(kRouteThreads) void route_kernel(const T* __restrict__ logits, RouteCall c, int per, int32_t* ids, float* weights, int32_t* offsets, int32_t* order, int32_t* blocks) {
    extern __shared__ int route_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int t0 = (int)blockIdx.x * per, t1 = min(t0 + per, c.tokens);
    for (int t = t0 + wave; t < t1; t += kRouteWaves) route_token<VPL>(logits, c, t, lane, ids, weights);
    __threadfence_block();
    __syncthreads();
    count_or_place(ids, t0 * c.top, t1 * c.top, c.experts, route_lds, offsets, order, blocks, wave, lane);
}

// Up to 32 pairs in all, one a lane (64 took 9.1 us where the sort below takes 6).  Its place is the number of pairs before it; every thread counts the pairs of experts below some.
template <int VPL, typename T>
__global__ __launch_bounds__(kRouteThreads) void route_few_kernel(const T* __restrict__ logits, RouteCall c, int32_t* __restrict__ ids, float* __restrict__ weights, int32_t* __restrict__ offsets,
                                                                  int32_t* __restrict__ order) {
    __shared__ int few[64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), pairs = c.tokens * c.top;
    int mine;
    if (c.tokens == 1) {
        mine = route_token<VPL>(logits, c, 0, lane, ids, weights);
    } else {
        for (int t = wave; t < c.tokens; t += (int)blockDim.x >> 6) {
            const int expert = route_token<VPL>(logits, c, t, lane, ids, weights);
            if (lane < c.top) few[t * c.top + lane] = expert;
        }
        __syncthreads();
        mine = few[lane];
    }
    if (lane >= pairs) mine = 0x7fffffff;
    if (wave == 0) {
        int place = 0;
        for (int i = 0; i < pairs; i++) {
            const int other = __builtin_amdgcn_readlane(mine, i);
            place += other < mine || (other == mine && i < lane);
        }
        if (lane < pairs) order[place] = lane;
    }
    for (int e0 = 0; e0 <= c.experts; e0 += (int)blockDim.x) {
        const int e = e0 + (int)threadIdx.x;
        int below = 0;
        for (int i = 0; i < pairs; i++) below += __builtin_amdgcn_readlane(mine, i) < e;
        if (e <= c.experts) offsets[e] = below;
    }
}

__global__ __launch_bounds__(kRouteThreads) void group_kernel(const int32_t* __restrict__ ids, int pairs, int experts, int per, int32_t* offsets, int32_t* order, int32_t* blocks) {
    extern __shared__ int route_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int from = (int)blockIdx.x * per, to = min(from + per, pairs);
    count_or_place(ids, from, to, experts, route_lds, offsets, order, blocks, wave, lane);
}

// The places of the pairs of each workgroup (per of them), after the counts of all.
__global__ __launch_bounds__(kRouteThreads) void place_kernel(const int32_t* __restrict__ ids, int pairs, int experts, int per, const int32_t* __restrict__ blocks, int32_t* __restrict__ offsets,
                                                              int32_t* __restrict__ order) {
    extern __shared__ int route_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), runs = experts + 1;
    int* const start = route_lds + kRouteWaves * runs;
    int* const before = start + runs;
    const int from = (int)blockIdx.x * per, to = min(from + per, pairs), first = ids[min(from + (int)threadIdx.x, to - 1)];
    for (int e = threadIdx.x; e < runs; e += kRouteThreads) start[e] = before[e] = 0;
    __syncthreads();
    // The counts of all workgroups and of those before this one: four experts a thread, as many threads for the same four as there are, each eight loads at a time
    // (4099 tokens, 128 experts, 257 workgroups: one expert a thread and eight loads at a time 11.4 us for the launch, this 7.5 us).
    const int quads = counts_stride(experts) / 4, shares = kRouteThreads / quads, blocks_all = (int)gridDim.x;  // 257 quads at most
    const int quad = (int)threadIdx.x % quads, share = (int)threadIdx.x / quads;
    if (share < shares) {
        int sum[4] = {}, mine[4] = {};
        for (int b0 = share; b0 < blocks_all; b0 += 8 * shares) {
            int4 v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = b0 + i * shares < blocks_all ? *(const int4*)(blocks + ((int64_t)(b0 + i * shares) * quads + quad) * 4) : int4{};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int own = b0 + i * shares < (int)blockIdx.x ? -1 : 0;
                sum[0] += v[i].x, sum[1] += v[i].y, sum[2] += v[i].z, sum[3] += v[i].w;
                mine[0] += v[i].x & own, mine[1] += v[i].y & own, mine[2] += v[i].z & own, mine[3] += v[i].w & own;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (quad * 4 + i < runs) {  // (behind the last expert's a row holds nothing that counts)
                atomicAdd(start + quad * 4 + i, sum[i]);
                atomicAdd(before + quad * 4 + i, mine[i]);
            }
        }
    }
    __syncthreads();
    exclusive_sums(start, runs, wave, lane);
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e < runs; e += kRouteThreads) offsets[e] = start[e];
    __syncthreads();
    for (int e = threadIdx.x; e < runs; e += kRouteThreads) start[e] += before[e];
    __syncthreads();
    place_pairs(ids, first, from, to, experts, route_lds, start, order, wave, lane);
}

// Tokens of a workgroup: all, up to two for each wavefront and 192 pairs; else one a wavefront and as many more as leave kRouteBlocks workgroups.  (A token after the other is 1 .. 2 us, a second launch 4: fp32
// tokens, 3 of 64 experts 32 6.9 us in one workgroup, 33 8.9 in two launches, 304 36.4 in one, 9.3 in two; 8 of 64 24 8.3 in one, 32 10.5, 33 9.6 in two.)
int64_t route_per(int64_t tokens, int top) { return tokens <= 2 * kRouteWaves && tokens * top <= 192 ? tokens : std::max<int64_t>(kRouteWaves, (tokens + kRouteBlocks - 1) / kRouteBlocks); }
// Pairs of a workgroup, where the experts are given.
int64_t group_per(int64_t pairs) { return pairs <= kRouteThreads ? pairs : std::max<int64_t>(kRouteThreads, (pairs + kRouteBlocks - 1) / kRouteBlocks); }
int64_t counts_bytes(int64_t blocks, int experts) { return blocks > 1 ? blocks * counts_stride(experts) * 4 : 0; }
size_t sort_lds(int experts) { return (size_t)(kRouteWaves + 2) * (experts + 1) * 4; }

template <int VPL, typename T>
hipError_t run_route(const T* logits, const RouteCall& c, int64_t per, int32_t* ids, float* weights, int32_t* offsets, int32_t* order, int32_t* blocks, hipStream_t s) {
    if ((int64_t)c.tokens * c.top <= 32) {
        route_few_kernel<VPL, T><<<dim3(1), dim3((unsigned)(64 * std::min(c.tokens, kRouteWaves))), 0, s>>>(logits, c, ids, weights, offsets, order);
        return hipGetLastError();
    }
    hipError_t e = allow_full_lds<route_kernel<VPL, T>>();
    if (e != hipSuccess) return e;
    route_kernel<VPL, T><<<dim3((unsigned)((c.tokens + per - 1) / per)), dim3(kRouteThreads), sort_lds(c.experts), s>>>(logits, c, (int)per, ids, weights, offsets, order, blocks);
    return hipGetLastError();
}
template <typename T>
hipError_t run_route(const T* logits, const RouteCall& c, int64_t per, int32_t* ids, float* weights, int32_t* offsets, int32_t* order, int32_t* blocks, hipStream_t s) {
    if (c.experts <= 64) return run_route<1>(logits, c, per, ids, weights, offsets, order, blocks, s);
    if (c.experts <= 128) return run_route<2>(logits, c, per, ids, weights, offsets, order, blocks, s);
    if (c.experts <= 256) return run_route<4>(logits, c, per, ids, weights, offsets, order, blocks, s);
    if (c.experts <= 512) return run_route<8>(logits, c, per, ids, weights, offsets, order, blocks, s);
    return run_route<16>(logits, c, per, ids, weights, offsets, order, blocks, s);
}

hipError_t run_places(const int32_t* ids, int64_t pairs, int experts, int64_t per, const int32_t* blocks, int32_t* offsets, int32_t* order, hipStream_t s) {
    hipError_t e = allow_full_lds<place_kernel>();
    if (e != hipSuccess) return e;
    place_kernel<<<dim3((unsigned)((pairs + per - 1) / per)), dim3(kRouteThreads), sort_lds(experts), s>>>(ids, (int)pairs, experts, (int)per, blocks, offsets, order);
    return hipGetLastError();
}

}  // namespace

int64_t route_workspace_bytes(int64_t tokens, int experts, int top) { return counts_bytes((tokens + route_per(tokens, top) - 1) / route_per(tokens, top), experts); }
int64_t group_workspace_bytes(int64_t pairs, int experts) { return counts_bytes((pairs + group_per(pairs) - 1) / group_per(pairs), experts); }

hipError_t launch_route_experts(const void* logits, int dtype, int64_t stride, int64_t tokens, int experts, int top, bool sigmoid, const float* bias, bool renormalize, float scale,
                                int32_t* ids, float* weights, int32_t* offsets, int32_t* order, void* workspace, hipStream_t s) {
    const RouteCall c{stride, (int)tokens, experts, top, sigmoid, renormalize, scale, bias};
    const int64_t per = route_per(tokens, top);
    int32_t* const blocks = per < tokens ? (int32_t*)workspace : nullptr;
    const hipError_t e = dtype == QMM_F32 ? run_route((const float*)logits, c, per, ids, weights, offsets, order, blocks, s) : run_route((const uint16_t*)logits, c, per, ids, weights, offsets, order, blocks, s);
    if (e != hipSuccess || !blocks) return e;
    return run_places(ids, tokens * top, experts, per * top, blocks, offsets, order, s);
}

hipError_t launch_group_experts(const int32_t* ids, int64_t pairs, int experts, int32_t* offsets, int32_t* order, void* workspace, hipStream_t s) {
    const int64_t per = group_per(pairs);
    int32_t* const blocks = per < pairs ? (int32_t*)workspace : nullptr;
    hipError_t e = allow_full_lds<group_kernel>();
    if (e != hipSuccess) return e;
    group_kernel<<<dim3((unsigned)((pairs + per - 1) / per)), dim3(kRouteThreads), sort_lds(experts), s>>>(ids, (int)pairs, experts, (int)per, offsets, order, blocks);
    e = hipGetLastError();
    if (e != hipSuccess || !blocks) return e;
    return run_places(ids, pairs, experts, per, blocks, offsets, order, s);
}

}  // namespace qmm
