// The experts' products with a few rows for each expert: the kernel for a few lhs rows (small_body.h), a workgroup's rows being some of an expert's pairs and its weights that expert's.  One launch, no workspace.
//
// Groups of up to MROWS pairs are counted over the experts (blockIdx.y; as many as there can be, those beyond the last leave at once), the tiles of 16 weight rows of each over blockIdx.x.  With one token
// every pair is a group and nothing is looked up.  What bounds it is the way to the first product and then the weights, as in the kernel that it is made of:
// one bf16 token, 8 of 64, 1024 x 2048 Q4_K gate and up 6.9 us (18.9 MB; 4 us to the first product); 16 fp32 tokens, 2 of 8, 14336 x 4096 Q5_K 75 us, 4.7 TB/s.
//
// The weighted sum of a token is a product too: the experts' super-blocks one after the other as one long K, each times its expert's weight, so that one launch ends
// with the token's results (a second launch, for the sum, is 2.5 us and the pairs' results written and read).
#include <math.h>

#include <algorithm>

#include "small_body.h"

namespace qmm {

namespace {

template <int ENC, int MROWS, typename AT, int MODE, int EX, bool PART>
__global__ __launch_bounds__(64 * kSmallWaves) void experts_small_kernel(MmMats mats, const AT* __restrict__ a, int m, int k, SmallCut cut, SmallExperts ex) {
    small_body<ENC, MROWS, AT, MODE, EX, PART>(mats, a, m, k, cut, ex);
}

struct EsPlan {
    int waves, groups, per, grid, chunk;
    size_t lds;
};
// tiles: of one group of rows; groups_y: groups of rows that are expected; nblk: super-blocks that a workgroup walks.  One round of workgroups if there are as many groups as expected, but no more than 16 tiles
// each: a group more than expected would otherwise be a round more (2 of 8 experts, 14336 x 4096 Q4_K, 16 fp32 rows 65 us, without the bound 46 or 90, with 8 tiles 71).
EsPlan es_plan(int encoding, int mrows, int64_t tiles, int64_t groups_y, int64_t nblk, bool part) {
    EsPlan p;
    // Groups of four rows whose tiles are many: two workgroups of half as many wavefronts on a compute unit, one of which multiplies while the other ends.  (8 of 64, 1024 x 4096 Q4_K gate and up, one bf16 row an
    // expert 49.7 -> 36.0 us, 2 of 8, 14336 x 4096 42.6 -> 37.4; Q6_K 77.5 -> 61.1.  With eight rows a group the lhs, narrowed for each of the groups of K, costs what that gains: Q6_K four rows an expert 86 -> 104.)
    const int most_waves = mrows == 4 && tiles * groups_y > 8 * (int64_t)compute_units() ? kSmallWaves / 2 : kSmallWaves;
    p.groups = (int)((nblk + most_waves - 1) / most_waves);
    p.waves = (int)((nblk + p.groups - 1) / p.groups);
    const int per_cu = std::max(1, kSmallWaves / p.waves);
    const int64_t places = std::max<int64_t>(1, (int64_t)compute_units() * per_cu / groups_y);
    const int64_t most = std::min<int64_t>((tiles + places - 1) / places, 16);
    p.grid = (int)((tiles + most - 1) / most);
    p.per = (int)((tiles + p.grid - 1) / p.grid);  // (small_body counts on `per` tiles or one less for every workgroup: (per - 1) grid < tiles)
    const int slot = encoding == QMM_Q4_0 || encoding == QMM_Q4_K ? SmallItem<QMM_Q4_K>::kSlot + (part ? 64 : 0) : encoding == QMM_Q5_K ? SmallItem<QMM_Q5_K>::kSlot : SmallItem<QMM_Q6_K>::kSlot;
    const int lr = mrows <= 4 ? 1 : mrows / 4, ring = p.waves * 2 * slot, bytes = (p.waves + (p.groups > 1 ? 1 : 0)) * lr * 256;
    p.chunk = std::min(std::min(p.per, 254), (kLdsPerCu / per_cu - ring) / bytes);
    p.lds = (size_t)ring + (size_t)p.chunk * bytes;
    return p;
}

template <int ENC, int MROWS, typename AT, int MODE, int EX, bool PART>
hipError_t run_part(const ExpertCall& c, const SmallExperts& ex, int64_t groups_y, int64_t expected, void* out, bool out_bf16, hipStream_t s) {
    const int tile = MODE == kSmallGated ? 8 : 16;
    const EsPlan p = es_plan(ENC, MROWS, (c.n + tile - 1) / tile, expected, (c.k + 255) / 256 * (EX == kSmallOverExperts ? ex.r.top : 1), PART);
    const hipError_t e = allow_full_lds<experts_small_kernel<ENC, MROWS, AT, MODE, EX, PART>>();
    if (e != hipSuccess) return e;
    MmMats mats{};
    for (int j = 0; j < kLanesMaxMats; j++) {
        mats.w[j] = c.w[j == 1 && c.gated ? 1 : 0];
        mats.out[j] = (float*)out;
        mats.n[j] = (int)c.n;
    }
    mats.count = 1;
    const SmallCut cut{p.per, p.grid, (uint32_t)p.waves | (uint32_t)p.chunk << 8 | (uint32_t)out_bf16 << 16 | (uint32_t)p.groups << 18};
    experts_small_kernel<ENC, MROWS, AT, MODE, EX, PART><<<dim3((unsigned)p.grid, (unsigned)groups_y), dim3((unsigned)(64 * p.waves)), p.lds, s>>>(mats, (const AT*)c.lhs, MROWS, (int)c.k, cut, ex);
    return hipGetLastError();
}
template <int ENC, int MROWS, typename AT, int MODE, int EX>
hipError_t run_small(const ExpertCall& c, const SmallExperts& ex, int64_t groups_y, int64_t expected, void* out, bool out_bf16, hipStream_t s) {
    if constexpr (ENC == QMM_Q4_0 && MROWS < 16) {  // (es_rows: no groups of 16 rows with partial super-blocks)
        if (c.k % 256) return run_part<ENC, MROWS, AT, MODE, EX, true>(c, ex, groups_y, expected, out, out_bf16, s);
    }
    return run_part<ENC, MROWS, AT, MODE, EX, false>(c, ex, groups_y, expected, out, out_bf16, s);
}
template <int ENC, int MROWS, typename AT>
hipError_t run_small(const ExpertCall& c, const SmallExperts& ex, int64_t groups_y, int64_t expected, void* out, bool out_bf16, hipStream_t s) {
    return c.gated ? run_small<ENC, MROWS, AT, kSmallGated, kSmallByExpert>(c, ex, groups_y, expected, out, out_bf16, s)
                   : run_small<ENC, MROWS, AT, kSmallPlain, kSmallByExpert>(c, ex, groups_y, expected, out, out_bf16, s);
}

// Experts that get a row, if none is preferred, and the rows that each of them gets, on average.
double es_with(const Routing& r) { return std::max(1.0, r.experts * (1.0 - pow(1.0 - std::min(1.0, (double)r.top / r.experts), (double)(r.pairs / r.top)))); }
double es_mean(const Routing& r) { return r.pairs / es_with(r); }
// Rows of a group.  us with 4 / 8 rows, 8 of 64 experts, 1024 x 2048 Q4_K: 2.3 rows an expert 17.9 / 18.9, 3.2 25.6 / 19.9; with 8 / 16: 6 27.4 / 33.1, 8 34.0 / 33.2.
int es_rows(const ExpertCall& c, const Routing& r, int64_t& expected) {
    const int64_t tokens = r.pairs / r.top, most = small_most_rows(c.lhs_dtype);
    if (tokens == 1) {
        expected = r.pairs;
        return 1;
    }
    const double mean = es_mean(r);
    const int rows = tokens <= 4 || mean <= 2.5 ? 4 : mean <= 6.5 || most == 8 || c.k % 256 ? 8 : 16;
    expected = std::max<int64_t>(1, (int64_t)(es_with(r) * std::max(1.0, mean / rows)));
    return rows;
}
int64_t es_groups(const Routing& r, int rows) { return r.pairs == r.top ? r.pairs : most_groups(r.pairs, r.experts, rows); }

template <int ENC>
hipError_t run_small(const ExpertCall& c, const SmallExperts& ex, void* out, bool out_bf16, hipStream_t s) {
    int64_t expected;
    const int rows = es_rows(c, ex.r, expected);
    const int64_t groups = es_groups(ex.r, rows);
    if (c.lhs_dtype == QMM_F32)
        return rows == 1   ? run_small<ENC, 1, float>(c, ex, groups, expected, out, out_bf16, s)
               : rows == 4 ? run_small<ENC, 4, float>(c, ex, groups, expected, out, out_bf16, s)
                           : run_small<ENC, 8, float>(c, ex, groups, expected, out, out_bf16, s);
    return rows == 1   ? run_small<ENC, 1, uint16_t>(c, ex, groups, expected, out, out_bf16, s)
           : rows == 4 ? run_small<ENC, 4, uint16_t>(c, ex, groups, expected, out, out_bf16, s)
           : rows == 8 ? run_small<ENC, 8, uint16_t>(c, ex, groups, expected, out, out_bf16, s)
                       : run_small<ENC, 16, uint16_t>(c, ex, groups, expected, out, out_bf16, s);
}
template <int ENC>
hipError_t run_sum(const ExpertCall& c, const SmallExperts& ex, void* out, bool out_bf16, hipStream_t s) {
    const int64_t tokens = ex.r.pairs / ex.r.top;
    return c.lhs_dtype == QMM_F32 ? run_small<ENC, 1, float, kSmallPlain, kSmallOverExperts>(c, ex, tokens, tokens, out, out_bf16, s)
                                  : run_small<ENC, 1, uint16_t, kSmallPlain, kSmallOverExperts>(c, ex, tokens, tokens, out, out_bf16, s);
}

bool es_takes(const ExpertCall& c) {
    if (kernel_disabled("experts_small")) return false;
    if ((c.k % 256 && (c.encoding != QMM_Q4_0 || c.k < 256)) || c.k > (1 << 20)) return false;
    const uintptr_t all = (uintptr_t)c.w[0] | (uintptr_t)c.expert_stride[0] | (c.gated ? (uintptr_t)c.w[1] | (uintptr_t)c.expert_stride[1] : 0);
    if (c.encoding == QMM_Q4_K || c.encoding == QMM_Q5_K) return (all & 15) == 0;
    if (all & 3) return false;
    return c.n * (c.encoding == QMM_Q4_0 ? c.k / 32 : c.k / 256) % 2 == 0;  // (loads of four bytes at least: the last block of a matrix has to end at a multiple of four)
}

}  // namespace

// Up to 8 rows an expert, or 12 where the GEMM unpacks more (bf16 rows but for Q4_K).  us, this kernel / the GEMM (with its preparation): 8 of 64 experts, 1024 x 2048, bf16 Q4_K 4 rows 19.8 / 28.0, 6 33.1 / 28.3,
// 12 33.3 / 29.1; Q6_K 8 45.3 / 40.3, 12 45.5 / 57.2; Q5_K 8 35.5 / 36.9, 12 35.8 / 43.8; fp32 Q4_K 8 29.5 / 31.3, 12 44.6 / 32.1; 2 of 8, 14336 x 4096, bf16 Q4_K 8 74 / 79, 12 105 / 88; Q6_K 12 112 / 136, 16 155 / 137.
// Q4_0: 8 of 64, 1024 x 2048 gate and up 8 bf16 rows 38.8 / 44.5; 1024 x 2080 (partial super-blocks) 6 47.1 / 48.0, 8 64.0 / 48.0.
bool experts_small_wanted(const ExpertCall& c, const Routing& r) {
    if (!es_takes(c) || es_mean(r) > (c.k % 256 ? 6.5 : c.lhs_dtype == QMM_F32 || c.encoding == QMM_Q4_K ? 8.0 : 12.0)) return false;
    int64_t expected;
    const int rows = es_rows(c, r, expected);
    return es_groups(r, rows) <= 65535;
}

hipError_t launch_experts_small(const ExpertCall& c, const Routing& r, void* out, bool out_bf16, hipStream_t s) {
    const SmallExperts ex{r, {c.expert_stride[0], c.expert_stride[1]}, c.lhs_top, nullptr, 0};
    switch (c.encoding) {
        case QMM_Q4_0: return run_small<QMM_Q4_0>(c, ex, out, out_bf16, s);
        case QMM_Q4_K: return run_small<QMM_Q4_K>(c, ex, out, out_bf16, s);
        case QMM_Q5_K: return run_small<QMM_Q5_K>(c, ex, out, out_bf16, s);
        default: return run_small<QMM_Q6_K>(c, ex, out, out_bf16, s);
    }
}

// One token, and a few that hardly share an expert (each reads the weights of its own): the share of the pairs that a router without preference sends to different experts.  us, products and sum / this, bf16 rows, Q4_K:
// 8 of 64, 2048 x 1024 2 tokens (0.94) 13.5 / 9.0, 4 (0.83) 15.7 / 11.8, 8 (0.66) 19.0 / 17.0; 2 of 128, 1536 x 1536 8 (0.95) 13.1 / 7.6; 4 of 16, 2048 x 1536 4 (0.68) 13.7 / 9.6; 2 of 8, 4096 x 14336 2 (0.88) 34.3 / 32.4,
// 3 (0.77) 49.1 / 52.7; 8 of 60, 7784 x 1024 4 (0.82) 31.1 / 30.0, 6 (0.72) 36.2 / 45.7.
bool experts_sum_small_wanted(const ExpertCall& c, const Routing& r) {
    if (!es_takes(c) || (c.k + 255) / 256 * r.top / kSmallWaves >= 0x1fff) return false;
    if (r.pairs == r.top) return true;
    const double share = es_with(r) / r.pairs;
    return share >= 0.8 || (share >= 0.6 && r.pairs * c.n * c.k <= (int64_t)48 << 20);
}

hipError_t launch_experts_sum_small(const ExpertCall& c, const Routing& r, const void* residual, int residual_dtype, void* out, bool out_bf16, hipStream_t s) {
    const SmallExperts ex{r, {c.expert_stride[0], c.expert_stride[1]}, c.lhs_top, residual, residual_dtype == QMM_BF16};
    switch (c.encoding) {
        case QMM_Q4_0: return run_sum<QMM_Q4_0>(c, ex, out, out_bf16, s);
        case QMM_Q4_K: return run_sum<QMM_Q4_K>(c, ex, out, out_bf16, s);
        case QMM_Q5_K: return run_sum<QMM_Q5_K>(c, ex, out, out_bf16, s);
        default: return run_sum<QMM_Q6_K>(c, ex, out, out_bf16, s);
    }
}

}  // namespace qmm
