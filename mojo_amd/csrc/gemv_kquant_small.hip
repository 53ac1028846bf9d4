// Q4_0, Q4_K, Q5_K and Q6_K with a few lhs rows (1 .. 16 bf16, 1 .. 8 fp32 a workgroup, up to four times as many side by side) on the matrix cores, K any multiple of 256: one launch, no workspace (groups of K side
// by side: a second launch and their sums in the workspace).
//
// Shape of the work.  A workgroup has as many wavefronts, up to 16, as divide the super-blocks of a row evenly into groups: wavefront w owns super-block
// w + waves g of group g (K = 4096: one group of 16; 14336: four of 14).  It converts the lhs columns of its super-block into matrix-core operands once a
// group, keeps them in 32 registers, and walks the workgroup's tiles of 16 weight rows with them.  The super-block of a tile's 16 rows (2.3 .. 3.8 KB) goes global -> LDS
// directly into a private ring of two slots, one item ahead of the one being multiplied: no wavefront waits for another before the end.  Partial results
// stay in LDS and are added in wavefront order, so their order depends on K only, not on N or on timing
// (the last bits of a row also on the rows beside it, whose values have a part in how it is scaled: small_lhs.h).
//
// Why 16 wavefronts with one super-block each (two before, eight wavefronts): an item is a chain LDS reads -> unpacking -> matrix cores of some 150 vector instructions, and with two
// wavefronts a SIMD most of it was waiting.  Why the rows of the lhs go where they go (row j to operand row 4 j mod 16, fp32 residuals in the rows between): a
// lane of the result holds operand rows 4 (lane / 16) + 0 .. 3, so with up to four rows every lane has one wanted result (two with fp32 residuals), and
// what is done to results (scales, sums, LDS) shrinks to a quarter.
//
// What bounds it: the way to the first product (launch, lhs from L2, conversion: some 4 us with four rows, 6 with sixteen), then memory (14336 x 4096, 4 bf16 rows: a tile of 16 rows, 37 .. 54 KB
// a compute unit, every 1.4 / 1.75 / 2.1 us).  Counters: vector instructions are issued in 0.57 .. 0.65 of a wavefront's life (403 of them in the 4.7 us of 4096 x 4096 with 4 fp32 rows, most for the lhs, and a SIMD's
// four wavefronts do it at the same time), 0.40 .. 0.46 of it is spent waiting, matrix cores are busy 0.09 .. 0.16.  us, the kernels before / this one, 14336 x 4096 4 bf16 rows, weights from memory: Q4_K 11.2 / 9.4, Q5_K 17.8 / 10.8, Q6_K 20.3 / 12.6; 16 bf16 rows
// 18.6 / 12.7, 17.5 / 13.9, 22.6 / 17.5; 4096 x 14336 4 fp32 rows 13.9 / 12.2, 22.7 / 13.9, 23.1 / 15.7; 2048 x 1024 4 bf16 rows 9.2 / 3.9.  Relative error, K = 4096, before / now: fp32 rows Q4_K
// 4.0e-7 / 1.1e-7, Q5_K 1.7e-7 / 1.2e-7, Q6_K 1.6e-7 / 1.0e-7; bf16 rows 2.5e-7 / 0.8e-7, 1.0e-7 / 0.85e-7, 0.97e-7 / 0.84e-7 (codes around their middle, residuals to nearest, super-blocks added in
// four chains).
//
// More rows than one workgroup takes: each streams all weights, the second one from its XCD's L2, which still beats preparing the lhs with a launch of its own where that launch and the next one's way to its first product
// are most of the time: 4096 x 4096 Q4_K 16 fp32 rows 11.7 / 9.2 us, 1024 x 14336 23.9 / 11.4 (rule and lines: qmm_api.hip).
//
// Arithmetic.  lhs: scaled by powers of two, then fp16 (see small_narrow; bf16 rows: one term; fp32 rows: hi part and residual, 22 bits).  Weights: integers sc * (q - mid) (Q4_K, Q5_K) or q (Q6_K) as fp16, so every product is exact and the sums are fp32.
//   Q4_K: a masked nibble is the subnormal q * 2^-24 (or 16 q * 2^-24), one packed multiply-add leaves sc * (q - 8) * 2^-18.
//   Q5_K: a byte permute puts nibble and fifth bit under 0x54: 64 + q; one packed multiply-add, (64 + q) * sc - 80 * sc, leaves sc * (q - 16) (exact: below 2^11).
//   Q6_K: the same with 96 taken off; sc * q may need 13 bits, so the scale multiplies the results of its 16 weights instead.
//   Q4_0 (an item is 16 rows x eight blocks): the lhs as Q8_0, quantised as any Q8_0 lhs here, int8 products of 16 (q - 8), whose sums over a block are exact; sum of (sum / 16) * (d_w d_a).
//   What codes around their middle leave out (Q4_K, Q5_K): mid * d * sc - dmin * mn times the sum of 32 lhs values, both as two fp16 terms, one more matrix product a super-block.
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "small_body.h"

namespace qmm {

// Wavefronts a SIMD that the compiler may aim at.  A launch has four, but for six it packs one and two bf16 rows of Q6_K into 80 registers where 90 keep an item's unpacking in flight: 4096 | 1024 | 1024
// x 4096 2 rows 8.4 / 7.8 us, 3664 | 3664 | 3664 x 1024 one row 5.3 / 4.95.
constexpr int small_simd_waves(int enc, int rows, int size, int mode) { return enc == QMM_Q6_K && rows <= 2 && size == 2 && mode == kSmallMats ? 5 : 8; }
template <int ENC, int MROWS, typename AT, int MODE>
__global__ __launch_bounds__(64 * kSmallWaves) __attribute__((amdgpu_waves_per_eu(4, small_simd_waves(ENC, MROWS, sizeof(AT), MODE)))) void gemv_kquant_small_mats_kernel(const MmMats mats, const AT* __restrict__ a, int m, int k, const SmallCut cut) {
    small_body<ENC, MROWS, AT, MODE>(mats, a, m, k, cut);
}

// The plain call: one matrix [n, k].  Twelve dwords of arguments.
template <int ENC, int MROWS, typename AT>
__global__ __launch_bounds__(64 * kSmallWaves) void gemv_kquant_small_kernel(const uint8_t* __restrict__ w, const AT* __restrict__ a, float* __restrict__ out, int n, int m, int k,
                                                                          int per, int stride, uint32_t packed) {
    MmMats mats;
    mats.w[0] = w;
    mats.out[0] = out;
    mats.n[0] = n;
    small_body<ENC, MROWS, AT, kSmallPlain>(mats, a, m, k, SmallCut{per, stride, packed});
}

namespace {

struct SmallPlan {
    int waves, groups, grid, parts, per, chunk, row_tiles;
    bool pairs;
    size_t lds;
};
// Groups of K: of its length only, so that results do not depend on what else a call has.
int small_groups(int64_t k) {
    const int groups = (int)((k / 256 + kSmallWaves - 1) / kSmallWaves);
    return groups == 3 ? 4 : groups;
}
// tiles: of 16 weight rows, gated: of eight of each matrix, or pairs of them (each = 2 items); parts: workgroups that share a tile, one group of K each; per: tiles of a workgroup, 0: as few as there are places for
SmallPlan small_plan(int encoding, int lhs_dtype, int64_t m, int64_t tiles, int64_t k, bool parts, int each = 1, int per = 0) {
    SmallPlan p;
    p.row_tiles = (int)((m + small_most_rows(lhs_dtype) - 1) / small_most_rows(lhs_dtype));
    m = std::min(m, small_most_rows(lhs_dtype));
    const int nblk = (int)(k / 256), groups = small_groups(k);
    p.groups = groups;
    p.waves = (nblk + groups - 1) / groups;
    p.parts = parts ? groups : 1;
    // one workgroup per compute unit (as many as 16 wavefronts allow with few each), all with the same number of tiles or one fewer
    const int per_cu = std::max(1, kSmallWaves / p.waves);
    const int64_t most = std::max<int64_t>(1, small_places(per_cu, p.row_tiles) / p.parts);
    p.per = per ? per : (int)((tiles + most - 1) / most);
    p.grid = (int)((tiles + p.per - 1) / p.per);
    const int slot = encoding == QMM_Q4_0 || encoding == QMM_Q4_K ? SmallItem<QMM_Q4_K>::kSlot : encoding == QMM_Q5_K ? SmallItem<QMM_Q5_K>::kSlot : SmallItem<QMM_Q6_K>::kSlot;
    // (as many items between two barriers as fit: a barrier after each, with two buffers, took Q6_K 28672 x 8192 with 16 rows from 65 to 92 us)
    const int lr = m <= 4 ? 1 : m <= 8 ? 2 : 4, ring = p.waves * 2 * slot, bytes = (p.waves + (groups > p.parts ? 1 : 0)) * lr * 256;
    p.chunk = std::min(std::min(each * p.per, 254), (kLdsPerCu / per_cu - ring) / bytes) / each * each;
    p.lds = (size_t)ring + (size_t)p.chunk * bytes;
    p.pairs = each == 2;
    return p;
}
// us: a tile of one group of K, the lhs of one
double small_item_us(int encoding) { return encoding == QMM_Q4_0 || encoding == QMM_Q4_K ? 1.4 : encoding == QMM_Q5_K ? 1.75 : 2.1; }
double small_convert_us(int encoding, int lhs_dtype, int64_t m) {
    return encoding == QMM_Q4_0 ? (m <= 2 ? 1.2 : m <= 4 ? 1.6 : m <= 8 ? 2.6 : 5.0)
           : lhs_dtype == QMM_F32 ? (m <= 2 ? 1.7 : m <= 4 ? 2.2 : 3.7) : (m <= 2 ? 1.5 : m <= 4 ? 1.7 : m <= 8 ? 3.0 : encoding == QMM_Q6_K ? 3.6 : 4.4);
}
// A gated pair: tiles with eight rows of each matrix, or pairs of whole ones?  By what the fullest compute unit gets, its workgroups' lhs and items one after the other.  The former may leave it an item less, but
// where several workgroups fit a compute unit they are more workgroups, and each converts the lhs: Q4_K 2816 x 1024 16 fp32 rows 6.5 / 7.3 us, Q4_0 4864 x 1024 8 fp32 rows 5.8 / 6.4 in pairs / halves.
// With more than four lhs rows a workgroup, pairs also where nothing is gained: half as many results to a wavefront's store is 2 .. 8 % there (9728 x 2560 16 fp32 rows Q4_0 13.6 / 14.4, 18944 x 3584
// 16 bf16 rows Q4_K 23.4 / 24.3); up to four rows, halves dealt like pairs (Q5_K 2816 x 1024 4 rows in pairs, halves, so dealt 4.5 / 4.3 / 4.15).  Over 460 calls, 1 .. 24 rows, 1.02 of the time of pairs at
// worst, 0.95 on average; always halves 0.96, up to 1.15.
SmallPlan small_gated_plan(int encoding, int lhs_dtype, int64_t m, int64_t n, int64_t k) {
    const SmallPlan halves = small_plan(encoding, lhs_dtype, m, (n + 7) / 8, k, false), pairs = small_plan(encoding, lhs_dtype, m, (n + 15) / 16, k, false, 2);
    const int64_t rows = std::min(m, small_most_rows(lhs_dtype));
    auto us = [&](const SmallPlan& p, int items) {
        const int64_t workgroups = ((int64_t)p.grid * p.row_tiles + compute_units() - 1) / compute_units();
        return workgroups * (small_convert_us(encoding, lhs_dtype, rows) + items * p.per * small_item_us(encoding));
    };
    if (rows > 4) return us(halves, 1) < 0.99 * us(pairs, 2) ? halves : pairs;
    return us(halves, 1) <= us(pairs, 2) ? halves : small_plan(encoding, lhs_dtype, m, (n + 7) / 8, k, false, 1, 2 * pairs.per);
}
// A K of several groups: a workgroup per (share of the tiles, group), whose results a launch of their own adds in group order, or all groups in each workgroup?
// The latter converts the lhs again for every group; both give the same bits.  us, walk / apart: Q4_K 1024 x 14336 4 bf16 rows 13.7 / 7.9, 4096 x 14336 2 bf16 rows
// 13.7 / 11.8, 8 fp32 rows 23.2 / 14.7; but two groups and many tiles, 28672 x 8192 4 bf16 rows 27.7 / 29.7, 8192 x 8192 11.5 / 12.1.
bool small_parts(int encoding, int lhs_dtype, int64_t m, int64_t n, int64_t k) {
    const int groups = small_groups(k);
    if (groups < 2) return false;
    const double item = small_item_us(encoding), convert = small_convert_us(encoding, lhs_dtype, m);
    const int64_t tiles = (n + 15) / 16;
    const SmallPlan w = small_plan(encoding, lhs_dtype, m, tiles, k, false), a = small_plan(encoding, lhs_dtype, m, tiles, k, true);
    const double walk = groups * ((w.per + w.chunk - 1) / w.chunk) * convert + groups * w.per * item;
    return convert + a.per * item + (a.per - 1) / a.chunk * 1.0 + 2.3 + 1.6e-6 * (4.0 * m * n * groups) < walk;
}

template <int ENC, int MROWS, typename AT>
hipError_t run_small(const MmMats& mats, const SmallPlan& p, const AT* a, int m, int k, bool gated, bool out_bf16, hipStream_t s) {
    const dim3 grid = p.row_tiles > 1 ? dim3(8, (unsigned)p.row_tiles, (unsigned)((p.grid * p.parts + 7) / 8)) : dim3((unsigned)p.grid, (unsigned)p.parts), block((unsigned)(64 * p.waves));
    const SmallCut cut{p.per, p.grid, (uint32_t)p.waves | (uint32_t)p.chunk << 8 | (uint32_t)out_bf16 << 16 | (uint32_t)(p.parts > 1) << 17 | (uint32_t)(p.parts > 1 ? 1 : p.groups) << 18 | (uint32_t)(p.row_tiles > 1) << 31};
    hipError_t e;
    if (gated && p.pairs) {
        if constexpr (MROWS > 4) {
            if ((e = allow_full_lds<gemv_kquant_small_mats_kernel<ENC, MROWS, AT, kSmallPairs>>()) != hipSuccess) return e;
            gemv_kquant_small_mats_kernel<ENC, MROWS, AT, kSmallPairs><<<grid, block, p.lds, s>>>(mats, a, m, k, cut);
        } else {
            return hipErrorInvalidValue;
        }
    } else if (gated) {
        if ((e = allow_full_lds<gemv_kquant_small_mats_kernel<ENC, MROWS, AT, kSmallGated>>()) != hipSuccess) return e;
        gemv_kquant_small_mats_kernel<ENC, MROWS, AT, kSmallGated><<<grid, block, p.lds, s>>>(mats, a, m, k, cut);
    } else if (mats.count > 1) {
        if ((e = allow_full_lds<gemv_kquant_small_mats_kernel<ENC, MROWS, AT, kSmallMats>>()) != hipSuccess) return e;
        gemv_kquant_small_mats_kernel<ENC, MROWS, AT, kSmallMats><<<grid, block, p.lds, s>>>(mats, a, m, k, cut);
    } else {
        if ((e = allow_full_lds<gemv_kquant_small_kernel<ENC, MROWS, AT>>()) != hipSuccess) return e;
        gemv_kquant_small_kernel<ENC, MROWS, AT><<<grid, block, p.lds, s>>>(mats.w[0], a, mats.out[0], mats.n[0], m, k, cut.per, cut.stride, cut.packed);
    }
    return hipGetLastError();
}

template <int ENC>
hipError_t run_small_rows(const MmMats& mats, const SmallPlan& p, const void* a, int lhs_dtype, int m, int k, bool gated, bool out_bf16, hipStream_t s) {
    if (lhs_dtype == QMM_F32) {
        const float* const f = (const float*)a;
        if (m == 1) return run_small<ENC, 1>(mats, p, f, m, k, gated, out_bf16, s);
        if (m <= 2) return run_small<ENC, 2>(mats, p, f, m, k, gated, out_bf16, s);
        if (m <= 4) return run_small<ENC, 4>(mats, p, f, m, k, gated, out_bf16, s);
        return run_small<ENC, 8>(mats, p, f, m, k, gated, out_bf16, s);
    }
    const uint16_t* const b = (const uint16_t*)a;
    if (m == 1) return run_small<ENC, 1>(mats, p, b, m, k, gated, out_bf16, s);
    if (m <= 2) return run_small<ENC, 2>(mats, p, b, m, k, gated, out_bf16, s);
    if (m <= 4) return run_small<ENC, 4>(mats, p, b, m, k, gated, out_bf16, s);
    if (m <= 8) return run_small<ENC, 8>(mats, p, b, m, k, gated, out_bf16, s);
    return run_small<ENC, 16>(mats, p, b, m, k, gated, out_bf16, s);
}

}  // namespace

bool gemv_kquant_small_supported(int encoding, int lhs_dtype, int64_t m, int64_t n, int64_t k, const void* w) {
    if (encoding != QMM_Q4_0 && encoding != QMM_Q4_K && encoding != QMM_Q5_K && encoding != QMM_Q6_K) return false;
    // (with the name of an encoding's older small-batch kernel this one goes too)
    if (kernel_disabled("kquant_small") || kernel_disabled(encoding == QMM_Q4_0 ? "q4_0_small" : encoding == QMM_Q4_K ? "q4k_mm" : encoding == QMM_Q5_K ? "q5k_mm" : "q6k_mm")) return false;
    if (m < 1 || m > small_most_rows(lhs_dtype) * 4 || n < 1 || n > 0x7fffff00 || k < 256 || k % 256 || k > (1 << 20)) return false;
    if (encoding == QMM_Q4_K || encoding == QMM_Q5_K) return ((uintptr_t)w & 15) == 0;
    if (encoding == QMM_Q4_0) return ((uintptr_t)w & 3) == 0;
    // (loads of four bytes at least: the last block of the matrix has to end at a multiple of four)
    return ((uintptr_t)w & 3) == 0 && n * (k / 256) % 2 == 0;
}

// What the fullest compute unit gets of a call whose workgroups walk K, a tile being 16 weight rows: small_tiles_wanted.
SmallLoad small_load(int lhs_dtype, int64_t m, int64_t n, int64_t k) {
    const SmallPlan p = small_plan(QMM_Q4_K, lhs_dtype, m, (n + 15) / 16, k, false);
    const int workgroups = ((int64_t)p.grid * p.row_tiles + compute_units() - 1) / compute_units();
    return {workgroups, workgroups * p.waves};
}

// What the parts of K of a plain call with few tiles take (without it a workgroup walks all of K: the same sums).
int64_t gemv_kquant_small_workspace_bytes(int encoding, int lhs_dtype, int64_t m, int64_t n, int64_t k) {
    return small_parts(encoding, lhs_dtype, m, n, k) ? small_groups(k) * m * n * 4 : 0;
}

namespace {
__global__ __launch_bounds__(256) void small_sum_bf16_kernel(const float* __restrict__ part, uint16_t* __restrict__ out, int64_t count, int parts) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    float v = 0.0f;
    for (int j = 0; j < parts; j++) v += part[j * count + i];
    out[i] = f2bf(v);
}
// The same for matrices that share a launch: matrix j has the values from end[j - 1] to end[j], and their shares at part[j], one after the other.
struct SmallSums {
    const float* part[kLanesMaxMats];
    float* out[kLanesMaxMats];
    int64_t end[kLanesMaxMats];
};
__global__ __launch_bounds__(256) void small_sum_mats_kernel(SmallSums sums, int parts) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= sums.end[kLanesMaxMats - 1]) return;
    const float* part = sums.part[0];
    float* out = sums.out[0];
    int64_t first = 0, end = sums.end[0];
#pragma unroll
    for (int j = 1; j < kLanesMaxMats; j++)
        if (i >= sums.end[j - 1]) part = sums.part[j], out = sums.out[j], first = sums.end[j - 1], end = sums.end[j];
    float v = 0.0f;
    for (int j = 0; j < parts; j++) v += part[j * (end - first) + i - first];
    out[i - first] = v;
}
}  // namespace
// out[i] = bf16(part[i] + part[count + i] + ...), in that order
hipError_t launch_sum_shares_bf16(const float* part, uint16_t* out, int64_t count, int shares, hipStream_t s) {
    small_sum_bf16_kernel<<<dim3((unsigned)((count + 255) / 256)), dim3(256), 0, s>>>(part, out, count, shares);
    return hipGetLastError();
}

// count matrices [ns[j], k] that share the lhs; gated: two of the same size, gate and up, outs[0] = silu(lhs gate^T) * (lhs up^T).  The caller has asked
// gemv_kquant_small_supported for each.  out_bf16: the outputs are bf16 arrays.  workspace: null, or (not gated) gemv_kquant_small_workspace_bytes with n = the sum of ns.
hipError_t launch_gemv_kquant_small(int encoding, const void* lhs, int lhs_dtype, int count, const void* const* ws, const int64_t* ns, float* const* outs, int64_t m, int64_t k,
                                    bool gated, bool out_bf16, void* workspace, hipStream_t s) {
    if (count < 1 || count > kLanesMaxMats || (gated && (count != 2 || ns[0] != ns[1]))) return hipErrorInvalidValue;
    MmMats mats;
    int64_t tiles = 0;
    for (int j = 0; j < kLanesMaxMats; j++) {
        const int i = std::min(j, count - 1);
        if (j < count) tiles += (ns[j] + 15) / 16;
        mats.w[j] = (const uint8_t*)ws[i];
        mats.out[j] = outs[gated ? 0 : i];
        mats.n[j] = (int)ns[i];
        mats.tile_end[j] = (int)tiles;
    }
    mats.count = count;
    int64_t all = 0;
    for (int j = 0; j < count; j++) all += ns[j];
    const bool parts = !gated && workspace && small_parts(encoding, lhs_dtype, m, all, k);
    SmallSums sums;
    int64_t values = 0;
    if (parts)
        for (int j = 0; j < kLanesMaxMats; j++) {
            sums.part[j] = mats.out[j] = (float*)workspace + values * small_groups(k);
            sums.out[j] = outs[std::min(j, count - 1)];
            if (j < count) values += m * ns[j];
            sums.end[j] = values;
        }
    const SmallPlan p = gated ? small_gated_plan(encoding, lhs_dtype, m, ns[0], k) : small_plan(encoding, lhs_dtype, m, tiles, k, parts);
    const bool store_bf16 = out_bf16 && !parts;
    hipError_t e = encoding == QMM_Q4_0   ? run_small_rows<QMM_Q4_0>(mats, p, lhs, lhs_dtype, (int)m, (int)k, gated, store_bf16, s)
                   : encoding == QMM_Q4_K ? run_small_rows<QMM_Q4_K>(mats, p, lhs, lhs_dtype, (int)m, (int)k, gated, store_bf16, s)
                   : encoding == QMM_Q5_K ? run_small_rows<QMM_Q5_K>(mats, p, lhs, lhs_dtype, (int)m, (int)k, gated, store_bf16, s)
                                          : run_small_rows<QMM_Q6_K>(mats, p, lhs, lhs_dtype, (int)m, (int)k, gated, store_bf16, s);
    if (e != hipSuccess || !parts) return e;
    if (count > 1) {  // (fp32 results: the callers with several matrices have no others)
        small_sum_mats_kernel<<<dim3((unsigned)((values + 255) / 256)), dim3(256), 0, s>>>(sums, p.parts);
        return hipGetLastError();
    }
    if (!out_bf16) return launch_sum_shares((const float*)workspace, outs[0], values, p.parts, s);
    return launch_sum_shares_bf16((const float*)workspace, (uint16_t*)outs[0], values, p.parts, s);
}

}  // namespace qmm
