// The experts' products for every shape: one wavefront takes one weight row (gated: one of gate and the same of up) of one expert for up to four of the expert's rows, a value at a time on the vector units.
//
// What the matrix-core kernels do not take goes here: weights at odd addresses, Q6_K rows with an odd number of blocks.  What bounds it is the unpacking, some twenty instructions a weight:
// 8 of 64 experts, 1024 x 2048 at an odd address, 1 / 16 / 64 bf16 tokens Q4_K 37 / 305 / 539 us, Q6_K 29 / 212 / 409, Q4_0 18 / 110 / 213.
// Q4_0: the lhs as Q8_0 codes and block scales (fp16, held as fp32), made by a launch in front; integer block dots.
// Also here: the weighted sum over the experts of a token, which ends the products of every kernel that leaves the pairs' results apart: 500 tokens, 8 experts,
// 2048 columns 7.6 us in a trace, 41 MB (5.4 TB/s, most of it from the caches).
#include <algorithm>

#include "experts.h"

namespace qmm {

namespace {

constexpr int kErRows = 4, kErWaves = 4;

// scale * code of weight i of a block, and what is taken off it
template <int ENC>
__device__ __forceinline__ float weight_of(const uint8_t* __restrict__ row, int k) {
    if constexpr (ENC == QMM_Q6_K) {
        const uint8_t* const b = row + (int64_t)(k >> 8) * Q6_K_BPB;
        const int i = k & 255, h = i >> 7, quarter = (i >> 5) & 3, at = i & 31;
        const int low = (b[64 * h + 32 * (quarter & 1) + at] >> (4 * (quarter >> 1))) & 15, high = (b[128 + 32 * h + at] >> (2 * quarter)) & 3;
        const float d = h2f((uint16_t)(b[208] | b[209] << 8));
        return d * (float)(int8_t)b[192 + (i >> 4)] * (float)((low | high << 4) - 32);
    } else {
        constexpr int kBpb = ENC == QMM_Q5_K ? Q5_K_BPB : Q4_K_BPB;
        const uint8_t* const b = row + (int64_t)(k >> 8) * kBpb;
        const int i = k & 255, j = i >> 5;
        const uint8_t* const s = b + 4;
        const int sc = j < 4 ? s[j] & 63 : (s[j + 4] & 15) | (s[j - 4] >> 6) << 4, mn = j < 4 ? s[j + 4] & 63 : (s[j + 4] >> 4) | (s[j] >> 6) << 4;
        int q = (b[kBpb - 128 + 32 * (j >> 1) + (i & 31)] >> (4 * (j & 1))) & 15;
        if constexpr (ENC == QMM_Q5_K) q |= ((b[16 + (i & 31)] >> j) & 1) << 4;
        const float d = h2f((uint16_t)(b[0] | b[1] << 8)), dmin = h2f((uint16_t)(b[2] | b[3] << 8));
        return fmaf(d * (float)sc, (float)q, -(dmin * (float)mn));
    }
}

struct ErArgs {
    const void* lhs;
    int lhs_top;
    const float* dscale;  // Q4_0: lhs = codes
    const uint8_t* w[2];
    int64_t stride[2], row_bytes;
    int gated, n, k;
    void* out;
    int out_bf16;
};

template <int ENC, typename AT>
__global__ __launch_bounds__(64 * kErWaves) void experts_rows_kernel(ErArgs a, Routing r) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int n = (int)blockIdx.x * kErWaves + wave;
    if (n >= a.n) return;
    for (int group = (int)blockIdx.y;; group += (int)gridDim.y) {
    const ExpertRows rows = find_rows<kErRows>(r, group, lane);
    if (rows.count == 0) return;
    int pair[kErRows];
#pragma unroll
    for (int j = 0; j < kErRows; j++) pair[j] = pair_at(r, rows.first + min(j, rows.count - 1));
    float sum[2][kErRows] = {};
    if (rows.expert < r.experts) {
        for (int h = 0; h <= a.gated; h++) {
            const uint8_t* const w = a.w[h] + rows.expert * a.stride[h] + n * a.row_bytes;
            if constexpr (ENC == QMM_Q4_0) {
                const int blocks = a.k / 32;
                for (int b = lane; b < blocks; b += 64) {
                    const uint8_t* const q = w + (int64_t)b * Q4_0_BPB;
                    const float d = h2f((uint16_t)(q[0] | q[1] << 8));
#pragma unroll
                    for (int j = 0; j < kErRows; j++) {
                        const int64_t at = (int64_t)(max(pair[j], 0) / a.lhs_top) * a.k + 32 * b;
                        const int8_t* const x = (const int8_t*)a.lhs + at;
                        int dot = 0;
                        for (int i = 0; i < 16; i++) dot += ((q[2 + i] & 15) - 8) * x[i] + ((q[2 + i] >> 4) - 8) * x[16 + i];
                        sum[h][j] = fmaf((float)dot, d * a.dscale[at >> 5], sum[h][j]);
                    }
                }
            } else {
                for (int k = lane; k < a.k; k += 64) {
                    const float v = weight_of<ENC>(w, k);
#pragma unroll
                    for (int j = 0; j < kErRows; j++) sum[h][j] = fmaf(v, load_f32((const AT*)a.lhs, (int64_t)(max(pair[j], 0) / a.lhs_top) * a.k + k), sum[h][j]);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kErRows; j++) {
        float y = wave_sum(sum[0][j]);
        if (a.gated) y = rows.expert < r.experts ? y / (1.0f + expf(-y)) * wave_sum(sum[1][j]) : 0.0f;
        if (lane == 0 && j < rows.count && pair[j] >= 0) {
            const int64_t at = (int64_t)pair[j] * a.n + n;
            if (a.out_bf16) ((uint16_t*)a.out)[at] = f2bf(y);
            else ((float*)a.out)[at] = y;
        }
    }
    }
}

// The lhs of Q4_0: codes and block scales, 32 lanes a block.
template <typename AT>
__global__ __launch_bounds__(256) void experts_quantize_kernel(const AT* __restrict__ x, int64_t blocks, int8_t* __restrict__ codes, float* __restrict__ dscale) {
    const int i = threadIdx.x & 31;
    for (int64_t block = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); block < blocks; block += (int64_t)gridDim.x * 8) {
        const float v = load_f32(x, block * 32 + i);
        float amax = fabsf(v);
#pragma unroll
        for (int mask = 16; mask; mask >>= 1) amax = fmaxf(amax, __shfl_xor(amax, mask, 32));
        uint16_t dh;
        const float id = q8_0_block_rule<true>(amax, dh);
        codes[block * 32 + i] = (int8_t)q8_0_code(v, id);
        if (i == 0) dscale[block] = h2f(dh);
    }
}

// Four results a thread (n a multiple of four, aligned rows) or one.
template <int V>
__global__ __launch_bounds__(256) void experts_combine_kernel(Routing r, const float* __restrict__ y, int n, const void* __restrict__ residual, int residual_bf16, void* __restrict__ out, int out_bf16) {
    const int64_t token = blockIdx.x;
    const int at = ((int)blockIdx.y * 256 + (int)threadIdx.x) * V;
    if (at >= n) return;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; i++) sum[i] = !residual ? 0.0f : residual_bf16 ? load_f32((const uint16_t*)residual, token * n + at + i) : load_f32((const float*)residual, token * n + at + i);
    for (int j = 0; j < r.top; j++) {
        const int64_t pair = token * r.top + j;
        const int id = r.ids[pair];
        if (id < 0 || id >= r.experts) continue;
        const float w = r.weights[pair];
        const float* const p = y + pair * n + at;
        if constexpr (V == 4) {
            const float4 v = *(const float4*)p;
            sum[0] = fmaf(w, v.x, sum[0]), sum[1] = fmaf(w, v.y, sum[1]), sum[2] = fmaf(w, v.z, sum[2]), sum[3] = fmaf(w, v.w, sum[3]);
        } else {
            sum[0] = fmaf(w, p[0], sum[0]);
        }
    }
    if (out_bf16) {
        uint16_t* const o = (uint16_t*)out + token * n + at;
        if constexpr (V == 4) *(uint2*)o = make_uint2(f2bf2(sum[0], sum[1]), f2bf2(sum[2], sum[3]));
        else o[0] = f2bf(sum[0]);
    } else {
        float* const o = (float*)out + token * n + at;
        if constexpr (V == 4) *(float4*)o = make_float4(sum[0], sum[1], sum[2], sum[3]);
        else o[0] = sum[0];
    }
}

}  // namespace

// Q4_0: codes, then block scales
int64_t experts_rows_workspace_bytes(const ExpertCall& c) { return c.encoding == QMM_Q4_0 ? (c.lhs_rows * c.k + 255) / 256 * 256 + c.lhs_rows * (c.k / 32) * 4 : 0; }

hipError_t launch_experts_rows(const ExpertCall& c, const Routing& r, void* out, bool out_bf16, void* workspace, hipStream_t s) {
    ErArgs a{c.lhs, c.lhs_top, nullptr, {c.w[0], c.w[1]}, {c.expert_stride[0], c.expert_stride[1]}, 0, c.gated, (int)c.n, (int)c.k, out, out_bf16};
    const dim3 grid((unsigned)((c.n + kErWaves - 1) / kErWaves), (unsigned)std::min<int64_t>(most_groups(r.pairs, r.experts, kErRows), 32768)), block(64 * kErWaves);
    if (c.encoding == QMM_Q4_0) {
        int8_t* const codes = (int8_t*)workspace;
        float* const dscale = (float*)(codes + (c.lhs_rows * c.k + 255) / 256 * 256);
        const int64_t blocks = c.lhs_rows * (c.k / 32);
        const dim3 groups((unsigned)std::min<int64_t>((blocks + 7) / 8, 1 << 20));  // (a grid has up to 2^32 threads)
        if (c.lhs_dtype == QMM_F32) experts_quantize_kernel<<<groups, dim3(256), 0, s>>>((const float*)c.lhs, blocks, codes, dscale);
        else experts_quantize_kernel<<<groups, dim3(256), 0, s>>>((const uint16_t*)c.lhs, blocks, codes, dscale);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        a.lhs = codes;
        a.dscale = dscale;
        a.row_bytes = c.k / 32 * Q4_0_BPB;
        experts_rows_kernel<QMM_Q4_0, float><<<grid, block, 0, s>>>(a, r);
        return hipGetLastError();
    }
#define QMM_ER(ENC, BPB)                                                                            \
    a.row_bytes = c.k / 256 * BPB;                                                                  \
    if (c.lhs_dtype == QMM_F32) experts_rows_kernel<ENC, float><<<grid, block, 0, s>>>(a, r);       \
    else experts_rows_kernel<ENC, uint16_t><<<grid, block, 0, s>>>(a, r)
    if (c.encoding == QMM_Q4_K) {
        QMM_ER(QMM_Q4_K, Q4_K_BPB);
    } else if (c.encoding == QMM_Q5_K) {
        QMM_ER(QMM_Q5_K, Q5_K_BPB);
    } else {
        QMM_ER(QMM_Q6_K, Q6_K_BPB);
    }
#undef QMM_ER
    return hipGetLastError();
}

hipError_t launch_experts_combine(const Routing& r, const float* y, int64_t n, const void* residual, int residual_dtype, void* out, bool out_bf16, hipStream_t s) {
    const int64_t tokens = r.pairs / r.top;
    const bool four = n % 4 == 0 && (((uintptr_t)y | (uintptr_t)out) & 15) == 0;
    const unsigned y_blocks = (unsigned)((n + (four ? 1024 : 256) - 1) / (four ? 1024 : 256));
    if (four) experts_combine_kernel<4><<<dim3((unsigned)tokens, y_blocks), dim3(256), 0, s>>>(r, y, (int)n, residual, residual_dtype == QMM_BF16, out, out_bf16);
    else experts_combine_kernel<1><<<dim3((unsigned)tokens, y_blocks), dim3(256), 0, s>>>(r, y, (int)n, residual, residual_dtype == QMM_BF16, out, out_bf16);
    return hipGetLastError();
}

}  // namespace qmm
