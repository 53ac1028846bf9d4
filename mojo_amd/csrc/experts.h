// What the experts' products share: the routing of a call and how a workgroup finds its rows.
#pragma once
#include "qmm_internal.h"

namespace qmm {

// A call's routing: pair p = top t + j is the j-th expert of token t.  order[offsets[e] .. offsets[e + 1]) are the pairs of expert e by rising number, behind the last those without an expert.
// Nothing that these arrays hold takes an access out of range: offsets are taken within 0 .. pairs, and what is no pair is left out.
struct Routing {
    const int32_t *offsets, *order, *ids;
    const float* weights;
    int pairs, top, experts;
};

// The rows of one expert that a workgroup takes: pairs order[first .. first + count); expert == routing.experts: those without one (their results are zeros).
struct ExpertRows {
    int expert, first, count;
};

__device__ __forceinline__ int offset_at(const Routing& r, int e) { return e > r.experts ? r.pairs : min(max(r.offsets[e], 0), r.pairs); }

// The same in scalar registers.  What a load in inline assembly takes as a scalar address must have been worked out there: five wait states lie between a vector instruction that writes a scalar
// register and a load that reads it, and the compiler, which moves an address over as late as it can, sees no load in the assembly and keeps none of them (such loads fault).
__device__ __forceinline__ ExpertRows uniform(const ExpertRows& x) {
    return {__builtin_amdgcn_readfirstlane(x.expert), __builtin_amdgcn_readfirstlane(x.first), __builtin_amdgcn_readfirstlane(x.count)};
}

// Number `group` of the groups of up to ROWS rows that the experts' runs are cut into, in the order of the experts; count 0: there are not so many.  One wavefront finds it, each lane with a
// share of the experts.  number(all): the wanted group's number, given how many there are.
template <int ROWS, typename F>
__device__ __forceinline__ ExpertRows find_rows_of(const Routing& r, int lane, F&& number) {
    const int per = r.experts / 64 + 1;  // (one run more than there are experts)
    int mine = 0;
    for (int i = 0, at = lane * per; i < per && at <= r.experts; i++, at++) mine += (max(offset_at(r, at + 1) - offset_at(r, at), 0) + ROWS - 1) / ROWS;
    int sum = mine;  // groups up to this lane's last run
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(sum, d);
        if (lane >= d) sum += o;
    }
    const int group = number(__shfl(sum, 63));
    const uint64_t beyond = group < 0 ? 0 : __ballot(sum > group);
    if (beyond == 0) return {0, 0, 0};
    const int owner = __builtin_ctzll(beyond);
    int left = group - (__shfl(sum, owner) - __shfl(mine, owner)), e = owner * per;
    for (; e <= r.experts; e++) {
        const int first = offset_at(r, e), count = max(offset_at(r, e + 1) - first, 0), groups = (count + ROWS - 1) / ROWS;
        if (left < groups) return left < 0 ? ExpertRows{0, 0, 0} : ExpertRows{e, first + left * ROWS, min(ROWS, count - left * ROWS)};  // (below 0: offsets of no sorted pairs, more groups than an int holds)
        left -= groups;
    }
    return {0, 0, 0};
}
template <int ROWS>
__device__ __forceinline__ ExpertRows find_rows(const Routing& r, int group, int lane) {
    return find_rows_of<ROWS>(r, lane, [&](int) { return group; });
}
// At most so many groups: every run but ends with one that may not be full.
inline int64_t most_groups(int64_t pairs, int experts, int rows) { return pairs / rows + experts + 1 < pairs ? pairs / rows + experts + 1 : pairs; }

// Pair number p of the run, -1 if it is none.
__device__ __forceinline__ int pair_at(const Routing& r, int place) {
    const int p = r.order[place];
    return p >= 0 && p < r.pairs ? p : -1;
}

// experts_route.hip
int64_t route_workspace_bytes(int64_t tokens, int experts, int top);
int64_t group_workspace_bytes(int64_t pairs, int experts);
hipError_t launch_route_experts(const void* logits, int dtype, int64_t stride, int64_t tokens, int experts, int top, bool sigmoid, const float* bias, bool renormalize, float scale,
                                int32_t* ids, float* weights, int32_t* offsets, int32_t* order, void* workspace, hipStream_t s);
hipError_t launch_group_experts(const int32_t* ids, int64_t pairs, int experts, int32_t* offsets, int32_t* order, void* workspace, hipStream_t s);

// One product by expert: rows x[pair / lhs_top] (lhs_top: the pairs of an lhs row, `top` or 1) times the weights w[0] (gated: and w[1]) of the pair's expert.
struct ExpertCall {
    int encoding;
    const void* lhs;
    int lhs_dtype, lhs_top;
    int64_t lhs_rows;
    const uint8_t* w[2];
    int64_t expert_stride[2];  // bytes between the matrices of neighbouring experts
    bool gated;
    int64_t n, k;
};
// out: fp32 or bf16 [pairs, n]
int64_t experts_rows_workspace_bytes(const ExpertCall& c);
hipError_t launch_experts_rows(const ExpertCall& c, const Routing& r, void* out, bool out_bf16, void* workspace, hipStream_t s);
// experts_gemm.hip
bool experts_gemm_supported(const ExpertCall& c, const Routing& r);
int64_t experts_gemm_workspace_bytes(const ExpertCall& c);
hipError_t launch_experts_gemm(const ExpertCall& c, const Routing& r, void* out, bool out_bf16, void* workspace, hipStream_t s);
// experts_small.hip: a few rows for each expert; the sum: one token, or a few that hardly share an expert
bool experts_small_wanted(const ExpertCall& c, const Routing& r);
hipError_t launch_experts_small(const ExpertCall& c, const Routing& r, void* out, bool out_bf16, hipStream_t s);
bool experts_sum_small_wanted(const ExpertCall& c, const Routing& r);
hipError_t launch_experts_sum_small(const ExpertCall& c, const Routing& r, const void* residual, int residual_dtype, void* out, bool out_bf16, hipStream_t s);
// out[t] = residual[t] + sum over j of weights[top t + j] y[top t + j], in that order (pairs without an expert left out); residual: null, fp32 or bf16
hipError_t launch_experts_combine(const Routing& r, const float* y, int64_t n, const void* residual, int residual_dtype, void* out, bool out_bf16, hipStream_t s);

// logprobs.hip
int64_t logprobs_workspace_bytes(int dtype, int64_t rows, int64_t vocab, int top);
hipError_t launch_logprobs(const void* logits, int dtype, int64_t stride, int64_t rows, int64_t vocab, const void* tokens, bool wide, int per_row, int top, float* chosen,
                           float* entropy, int32_t* top_ids, float* top_values, void* workspace, hipStream_t s);

}  // namespace qmm
