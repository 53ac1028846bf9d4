// The kernel for a few lhs rows (gemv_kquant_small.hip, which says how it works and why; experts_small.hip).
#pragma once
#include <algorithm>
#include <type_traits>

#include "experts.h"
#include "small_lhs.h"

namespace qmm {

namespace {

constexpr int kSmallWaves = 16;

// The item of a wavefront: 16 rows of one super-block.  kRow: bytes of a row in LDS; Q6_K blocks lie at even addresses, loads to LDS want multiples of
// four: 212 bytes from the last such address on, the last 16 of them as a piece of their own (which overlaps the one before), and one piece of padding that
// spreads the rows over the banks.
template <int ENC>
struct SmallItem {
    static constexpr int kBpb = ENC == QMM_Q4_0 ? 8 * Q4_0_BPB : ENC == QMM_Q4_K ? Q4_K_BPB : ENC == QMM_Q5_K ? Q5_K_BPB : Q6_K_BPB;  // of 256 columns
    static constexpr int kRow = ENC == QMM_Q6_K ? 240 : kBpb, kRowPieces = kRow / 16, kPieces = 16 * kRowPieces, kLoads = (kPieces + 63) / 64, kSlot = 16 * kRow;
    static_assert(4 * kSmallPlane + 16 <= kSlot, "four planes of lhs rows and their scales fit a ring slot");
};

enum { kSmallPlain = 0, kSmallMats = 1, kSmallGated = 2, kSmallPairs = 3 };

}  // namespace

// By expert (experts_small.hip).  kSmallByExpert: a workgroup's lhs rows are some of the pairs of one expert (blockIdx.y counts groups of up to MROWS of them), its weights that expert's; what would be
// rows of the lhs and of the results are those of the pairs.  kSmallOverExperts: one token (blockIdx.y), whose experts follow each other as if they were one long K, super-block by super-block, each
// times its expert's weight: the weighted sum in one launch.
enum { kSmallNoExperts = 0, kSmallByExpert = 1, kSmallOverExperts = 2 };
struct SmallExperts {
    Routing r;
    int64_t stride[2];
    int lhs_top;
    const void* residual;  // kSmallOverExperts
    int residual_bf16;
};

// MROWS: lhs rows of a workgroup, 1, 2, 4, 8 or 16 (rows past m repeat the last one and their results are dropped); more go side by side, in workgroups of their own.
// MODE: one matrix; several that share the lhs (their tiles numbered through); gate and up (result silu(gate) * up), eight rows of each in a tile, or a tile of gate and one of up after the other.
struct SmallCut {
    int per, stride;  // tiles (pairs of them) of a workgroup at most, workgroups across the tiles
    uint32_t packed;  // wavefronts; << 8: items (tile of a matrix, or of both) of a workgroup whose partial results fit LDS together; << 16: bf16 results; << 17: a group of K per workgroup; << 18: groups of a workgroup; << 31: several tiles of lhs rows
};
// PART (Q4_0, experts): K is no multiple of 256 (but no less).  The last super-block of a row begins 256 columns before its end; of the lhs, what the one before has too is taken as zeros there.  Rows and
// super-blocks begin at even addresses, loads to LDS want multiples of four: a row's nine pieces from the last such address on, and four bytes more that a row which begins two bytes later needs.
template <int ENC, int MROWS, typename AT, int MODE, int EX = kSmallNoExperts, bool PART = false>
__device__ __forceinline__ void small_body(const MmMats& mats, const AT* __restrict__ a, int m, int k, const SmallCut& cut, const SmallExperts& ex = SmallExperts{}) {
    using I = SmallItem<ENC>;
    constexpr bool kQ8 = ENC == QMM_Q4_0;                   // the lhs as Q8_0 codes and block scales
    constexpr int PL = sizeof(AT) == 4 && !kQ8 ? 2 : 1;     // operand rows of an lhs row
    constexpr int LR = MROWS <= 4 ? 1 : MROWS / 4;          // lhs rows of a lane's results: lane / 16 + 4 j
    constexpr int RN = LR * PL;
    constexpr int kPass = std::min(MROWS, 4 / PL);          // lhs rows that change lanes together
    static_assert(RN <= 4, "operand rows");
    static_assert(!PART || (kQ8 && EX != kSmallNoExperts), "partial super-blocks");
    constexpr int kSlot = I::kSlot + (PART ? 64 : 0), kLoads = I::kLoads + (PART ? 1 : 0);
    constexpr bool kMin = ENC == QMM_Q4_K || ENC == QMM_Q5_K;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    // (what follows from the launch comes as arguments: the compiler fetches blockDim and gridDim with a vector load and waits for it)
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (int)(cut.packed & 0xffu), chunk = (int)(cut.packed >> 8) & 0xff, per = cut.per, stride = cut.stride;
    const bool out_bf16 = (cut.packed >> 16) & 1, apart = (cut.packed >> 17) & 1;
    const int nn = lane & 15, kg = lane >> 4;
    const int row_blocks = PART ? (k + 255) >> 8 : k >> 8, nblk = EX == kSmallOverExperts ? row_blocks * ex.r.top : row_blocks, groups = (int)(cut.packed >> 18) & 0x1fff;
    int share = (int)blockIdx.x, part = (int)blockIdx.y, row0 = 0;  // this workgroup's tiles, group of K, first lhs row
    if (MROWS == small_rows<AT>() && (cut.packed >> 31)) {
        // several tiles of lhs rows: those that read the same weights side by side (blockIdx.y) on one XCD (ids congruent mod 8), every XCD the same number of them
        row0 = (int)blockIdx.y * MROWS, share = (int)blockIdx.z * 8 + (int)blockIdx.x, part = apart ? share / stride : 0;
        share -= part * stride;
        if (share >= stride || (apart && part * waves >= nblk)) return;  // (the whole workgroup)
    }
    ExpertRows er{0, 0, 0};
    int lhs_rows[MROWS], my_pairs[LR];  // the rows' places in the lhs; the pairs of this lane's results
    int token_ids = -1;               // kSmallOverExperts: lane j: the token's j-th expert, -1: none, and its weight
    float token_weights = 0.0f;
    if constexpr (EX == kSmallByExpert) {
        part = (int)blockIdx.z;  // (0; the compiler, told so, takes the loop over the groups of K apart and spills)
        er = ex.r.pairs == ex.r.top ? ExpertRows{ex.r.ids[blockIdx.y], (int)blockIdx.y, 1} : find_rows<MROWS>(ex.r, (int)blockIdx.y, lane);  // (one token: a group for each pair, in their order)
        const bool one = ex.r.pairs == ex.r.top;
        er = uniform(er);
        if (er.count == 0) return;
        m = er.count;
        const int listed = one ? er.first : pair_at(ex.r, er.first + min(lane & 15, er.count - 1));
        const int places = max(listed, 0) / ex.lhs_top;
#pragma unroll
        for (int j = 0; j < MROWS; j++) lhs_rows[j] = __builtin_amdgcn_readlane(places, j);
#pragma unroll
        for (int j = 0; j < LR; j++) my_pairs[j] = __shfl(listed, kg + 4 * j);
        if (er.expert < 0 || er.expert >= ex.r.experts) {  // pairs without an expert: zeros
            const int first = share * (MODE == kSmallGated ? 8 : 16), step = stride * (MODE == kSmallGated ? 8 : 16);
            for (int n0 = first; n0 < mats.n[0]; n0 += step)
                for (int i = tid; i < 16 * er.count; i += 64 * waves) {
                    const int pair = one ? er.first : pair_at(ex.r, er.first + (i >> 4)), n = n0 + (i & 15);
                    if (pair < 0 || (i & 15) >= (MODE == kSmallGated ? 8 : 16) || n >= mats.n[0]) continue;
                    if (out_bf16) ((uint16_t*)mats.out[0])[(int64_t)pair * mats.n[0] + n] = 0;
                    else mats.out[0][(int64_t)pair * mats.n[0] + n] = 0.0f;
                }
            return;
        }
    }
    if constexpr (EX == kSmallOverExperts) {
        part = (int)blockIdx.z;
        const int64_t pair = (int64_t)blockIdx.y * ex.r.top + min(lane, ex.r.top - 1);
        const int id = ex.r.ids[pair];
        token_ids = id < ex.r.experts ? max(id, -1) : -1;
        token_weights = ex.r.weights[pair];
    }
    // super-block sb of a row of the lhs; kSmallOverExperts: of the row that the token's expert sb / row_blocks gets
    auto lhs_at = [&](int j, int sb) __attribute__((always_inline)) -> const AT* {
        if constexpr (EX == kSmallByExpert) return a + (int64_t)lhs_rows[j] * k + (PART ? min(sb * 256, k - 256) : sb * 256);
        if constexpr (EX == kSmallOverExperts) {
            const int of = sb / row_blocks;
            return a + (int64_t)(((int)blockIdx.y * ex.r.top + of) / ex.lhs_top) * k + (PART ? min((sb - of * row_blocks) * 256, k - 256) : (sb - of * row_blocks) * 256);
        }
        return a + (int64_t)min(row0 + j, m - 1) * k + sb * 256;
    };
    // One group per workgroup (then groups is 1, and the operands of the first conversion serve every item), or all of them.  (A flag or a comparison of the group's number instead, as `groups > 1` below, took Q6_K 1184 x 1024
    // with 33 rows from 4.95 to 5.11 us.)
    const int g_first = apart ? part : 0, g_end = apart ? g_first + 1 : groups;
    const uint32_t row_bytes = PART ? (uint32_t)(k / 32 * Q4_0_BPB) : (uint32_t)(row_blocks * I::kBpb);
    uint8_t* const ring = smem + wave * (2 * kSlot);
    const uint32_t ring_lds = lds_address(ring);
    float* const accs = (float*)(smem + waves * (2 * kSlot));  // [chunk][waves][LR][64]
    float* const totals = accs + chunk * waves * LR * 64;  // [chunk][LR][64], with more than one group
    // Weight rows of a matrix in a tile.  Gated, eight of gate and the same eight of up: a workgroup has results whole with half as many of them.  14336 x 4096 4 bf16 rows: seven such tiles for each
    // of 256 compute units, where 896 pairs of whole tiles were four (eight tiles) for each of 224, 15.3 -> 13.9 us; Q6_K 13824 x 5120 28.8 -> 26.9, Q4_K 1000 x 4096 3 rows 6.9 -> 5.8.  The same sums.
    // Pairs of whole tiles are left to small_gated_plan's choice.
    constexpr int kTile = MODE == kSmallGated ? 8 : 16, kEach = MODE == kSmallPairs ? 2 : 1;  // kEach: items that make a result
    const int ntiles = MODE == kSmallMats ? mats.tile_end[kLanesMaxMats - 1] : (mats.n[0] + kTile - 1) / kTile;
    const int my_items = kEach * (share + (per - 1) * stride < ntiles ? per : per - 1);  // (the grid has no workgroup without a tile)

    // item i of the workgroup: its matrix, and the first row there
    auto matrix_of = [&](int i, int& n0, int& n) __attribute__((always_inline)) {
        const int tile = share + i / kEach * stride;
        int j = 0;
        if constexpr (MODE == kSmallMats) {  // (entries past the last repeat it)
#pragma unroll
            for (int i = 0; i + 1 < kLanesMaxMats; i++) j += tile >= mats.tile_end[i] ? 1 : 0;
        }
        n0 = (MODE == kSmallMats && j ? tile - mats.tile_end[j - 1] : tile) * kTile;
        if constexpr (MODE == kSmallPairs) j = i & 1;
        n = mats.n[j];
        return j;
    };
    // piece p = lane + 64 i of an item: row p / kRowPieces
    uint32_t full[I::kLoads];  // byte offset of the piece (Q6_K, PART: of its row) in a tile that lies inside the matrix
    uint32_t at_row = 0;       // Q6_K, PART: where it begins in the row, eight bits each
#pragma unroll
    for (int i = 0; i < I::kLoads; i++) {
        const int p = min(lane + 64 * i, I::kPieces - 1), pr = p / I::kRowPieces, pc = p - pr * I::kRowPieces;
        full[i] = (uint32_t)(pr % kTile) * row_bytes + (ENC == QMM_Q6_K || PART ? 0u : 16u * (uint32_t)pc);
        if constexpr (ENC == QMM_Q6_K) at_row |= (pc < 13 ? 16u * (uint32_t)pc : 196u) << (8 * i);
        if constexpr (PART) at_row |= 16u * (uint32_t)pc << (8 * i);
    }
    // PART: where super-block sb of a row begins
    auto window = [&](int sb) __attribute__((always_inline)) { return min((uint32_t)sb * (uint32_t)I::kBpb, row_bytes - (uint32_t)I::kBpb); };
    auto issue = [&](int sb, int item, int slot) {
        int n0, n;
        const int j = matrix_of(item, n0, n);
        int64_t expert_at = 0;
        if constexpr (EX == kSmallByExpert) expert_at = er.expert * ex.stride[j];
        if constexpr (EX == kSmallOverExperts) {
            const int of = sb / row_blocks;
            sb -= of * row_blocks;
            expert_at = max(__builtin_amdgcn_readlane(token_ids, of), 0) * ex.stride[0];
        }
        const uint8_t* const base = mats.w[j] + expert_at + (int64_t)n0 * row_bytes + (ENC == QMM_Q6_K || PART ? 0 : sb * I::kBpb);
        const uint8_t* const base2 = MODE == kSmallGated ? mats.w[1] + (base - mats.w[0]) + (EX == kSmallByExpert ? er.expert * (ex.stride[1] - ex.stride[0]) : 0) : base;
        const int last = n - 1 - n0;  // rows past the matrix repeat its last row (their results are dropped)
#pragma unroll
        for (int i = 0; i < I::kLoads; i++) {
            uint32_t off = full[i];
            if (last < kTile - 1) {  // (the last tile of a ragged matrix only)
                const int pr = min(lane + 64 * i, I::kPieces - 1) / I::kRowPieces % kTile;
                off -= (uint32_t)(pr - min(pr, last)) * row_bytes;
            }
            if constexpr (ENC == QMM_Q6_K) off = ((off + (uint32_t)(sb * Q6_K_BPB)) & ~3u) + ((at_row >> (8 * i)) & 0xffu);
            if constexpr (PART) off = ((off + window(sb)) & ~3u) + ((at_row >> (8 * i)) & 0xffu);
            if (i < I::kLoads - 1 || I::kPieces % 64 == 0 || lane < I::kPieces - 64 * (I::kLoads - 1)) {
                const uint32_t to = ring_lds + slot * kSlot + i * 1024;
                constexpr int kGate = 8 * I::kRowPieces;  // pieces of the first of two matrices
                if (MODE != kSmallGated || 64 * (i + 1) <= kGate) small_stream16(off, base, to);
                else if (64 * i >= kGate) small_stream16(off, base2, to);
                else load16_to_lds_once((lane + 64 * i < kGate ? base : base2) + off, to);
            }
        }
        if constexpr (PART) {
            if (lane < 16) {
                const uint32_t at = (uint32_t)min(lane % kTile, last) * row_bytes + window(sb);
                load4_to_lds((MODE != kSmallGated || lane < 8 ? base : base2) + (at & 2u ? (at & ~3u) + I::kBpb : at & ~3u), ring_lds + slot * kSlot + I::kSlot);
            }
        }
    };

    // ---- lhs operands of the wavefront's super-block.  Operand row nn: lhs row nn / 4 + 4 j, hi part or (fp32) residual, j and part by nn % 4.
    // Q4_K, Q5_K: fragment (p, h) of lane quarter kg holds columns 64 kg + 32 h + 8 p + (0 .. 7; Q4_K in the order 0,2,1,3,4,6,5,7); Q6_K: fragment g holds 16 g + 4 kg + 0 .. 3.
    // Q4_0: block b of lane quarter kg holds the codes of columns 4 kg .. + 3 and 16 + 4 kg .. + 3; block scales of this lane's results, two fp16 numbers a register.
    half8 fa[kMin ? 4 : 1][2], fs;
    ks_half4 fq[ENC == QMM_Q6_K ? 16 : 1];
    u32x2 fc[kQ8 ? 8 : 1];
    u32x4 fd[kQ8 ? LR : 1];
    float bs[LR];  // inverse lhs scales of this lane's results
#pragma unroll
    for (int b = 0; b < (kQ8 ? 8 : 1); b++) fc[b] = u32x2{0u, 0u};
#pragma unroll
    for (int j = 0; j < (kQ8 ? LR : 1); j++) fd[j] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int p = 0; p < (kMin ? 4 : 1); p++) fa[p][0] = fa[p][1] = pack4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int g = 0; g < (ENC == QMM_Q6_K ? 16 : 1); g++) fq[g] = ks_half4{0, 0, 0, 0};
    fs = pack4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int j = 0; j < LR; j++) bs[j] = 0.0f;
    typedef typename std::conditional<sizeof(AT) == 4, u32x4, u32x2>::type xraw_t;
    // xr: columns 4 lane .. 4 lane + 3 of every lhs row; area: a free ring slot
    auto narrow = [&](const xraw_t (&xr)[MROWS], uint8_t* area) __attribute__((always_inline)) {
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));  // (what is computed from it here is not kept in registers between the groups)
        const int nn = lane & 15, kg = lane >> 4, my_row = (nn >> 2) + 4 * ((nn & 3) / PL), my_part = (nn & 3) % PL;
        if constexpr (kQ8) {
#pragma unroll
            for (int r0 = 0; r0 < MROWS; r0 += kPass) {
                small_quantize<kPass, EX != kSmallNoExperts>(xr, r0, area, lane);
                asm volatile("" ::: "memory");  // (scales are written as 16-bit numbers and read as vectors: not to be reordered)
                __builtin_amdgcn_wave_barrier();
                if ((nn & 3) < RN && my_row >= r0 && my_row < r0 + kPass) {
                    const uint8_t* const pl = area + (my_row - r0) * kSmallCodes;
#pragma unroll
                    for (int b = 0; b < 8; b++) fc[b] = *(const u32x2*)(pl + 32 * b + 8 * kg);
                }
#pragma unroll
                for (int j = 0; j < LR; j++)
                    if (kg + 4 * j >= r0 && kg + 4 * j < r0 + kPass) fd[j] = *(const u32x4*)(area + (kg + 4 * j - r0) * kSmallCodes + 256);
            }
        } else {
            float* const scales = (float*)(area + 4 * kSmallPlane);
            constexpr int kTop = kMin ? 9 : 14;
            float common = 1.0f;
            if constexpr (PL == 2) common = small_common_scale<kTop>(xr);
#pragma unroll
            for (int r0 = 0; r0 < MROWS; r0 += kPass) {
                const float inverse = small_narrow<PL, kPass, ENC == QMM_Q4_K ? kSmallOrderK : kSmallOrderPlain, kTop>(xr, r0, common, area, scales, lane);
                __builtin_amdgcn_wave_barrier();
                if ((nn & 3) < RN && my_row >= r0 && my_row < r0 + kPass) {
                    const uint8_t* const pl = area + ((my_row - r0) * PL + my_part) * kSmallPlane;
                    if constexpr (ENC == QMM_Q6_K) {
#pragma unroll
                        for (int g = 0; g < 16; g++) fq[g] = *(const ks_half4*)(pl + 32 * g + 8 * kg);
                    } else {
#pragma unroll
                        for (int p = 0; p < 4; p++) {
                            fa[p][0] = *(const half8*)(pl + 128 * kg + 16 * p);
                            fa[p][1] = *(const half8*)(pl + 128 * kg + 64 + 16 * p);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < LR; j++)
                    if (kg + 4 * j >= r0 && kg + 4 * j < r0 + kPass) bs[j] = inverse == 0.0f ? scales[kg + 4 * j - r0] : inverse;
            }
        }
        if constexpr (kMin) {
            // Sums of the operand rows over 32 columns on the matrix cores: column j < 4 of the product is sub-block 2 j (the lane quarter kg = j supplies the ones),
            // column 4 + j sub-block 2 j + 1.  Through LDS they come to the lane that supplies them: (row nn, sub-blocks 2 kg, 2 kg + 1), as two fp16 terms.
            const uint32_t e0 = nn == kg ? 0x3C003C00u : 0u, e1 = nn == kg + 4 ? 0x3C003C00u : 0u;
            const half8 ones0 = pack4(e0, e0, e0, e0), ones1 = pack4(e1, e1, e1, e1);
            ks_float4 S = {0.f, 0.f, 0.f, 0.f}, S1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = 0; p < 4; p++) {
                S = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[p][0], ones0, S, 0, 0, 0);
                S1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[p][1], ones1, S1, 0, 0, 0);
            }
            S += S1;
            float* const st = (float*)area;
            __builtin_amdgcn_wave_barrier();
            if (nn < 8) {
#pragma unroll
                for (int r = 0; r < RN; r++) st[(4 * kg + r) * 9 + nn] = S[r];
            }
            __builtin_amdgcn_wave_barrier();
            const float s0 = (nn & 3) < RN ? st[nn * 9 + kg] : 0.0f, s1 = (nn & 3) < RN ? st[nn * 9 + 4 + kg] : 0.0f;
            const half2v sh = to_half2(s0, s1), sl = to_half2(fmaf((float)sh.x, -1.0f, s0), fmaf((float)sh.y, -1.0f, s1));
            const uint32_t h = __builtin_bit_cast(uint32_t, sh), l = __builtin_bit_cast(uint32_t, sl);
            fs = pack4((h & 0xffffu) | (l << 16), h, (l >> 16) | (h & 0xffff0000u), 0u);  // (sh0, sl0), (sh0, sh1), (sl1, sh1)
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the operands are in registers before the next item's load may overwrite the slot
    };
    const uint32_t a_lane = 4 * (uint32_t)sizeof(AT) * lane;
    // PART: the columns of a row's last super-block that the one before has too
    auto leave_out = [&](xraw_t (&xr)[MROWS], int sb) __attribute__((always_inline)) {
        if (sb % row_blocks == row_blocks - 1 && 4 * lane < 256 * row_blocks - k) {
#pragma unroll
            for (int j = 0; j < MROWS; j++) xr[j] = xraw_t{};
        }
    };

    // first group: the lhs, then the first weights, which stay on their way while the lhs is converted.  (Straight-line code: nothing may move a register that such a load has
    // not filled yet.  A wavefront without a super-block, in the last group, takes the last one and drops it.)
    int slot = 0;
    {
        xraw_t xr[MROWS];
        const int sb = min(g_first * waves + wave, nblk - 1);
#pragma unroll
        for (int j = 0; j < MROWS; j++) hidden_load(xr[j], a_lane, lhs_at(j, sb));
        issue(sb, 0, 0);
        wait_vmcnt<kLoads>();
#pragma unroll
        for (int j = 0; j < MROWS; j++) tie(xr[j]);
        if constexpr (PART) leave_out(xr, sb);
        narrow(xr, ring + kSlot);
    }
    // (constants of the unpack in vector registers: an and-or in one instruction takes no literal and one scalar at most)
    uint32_t m_low = ENC == QMM_Q5_K ? 0x01010101u : 0x03030303u, c54 = 0x54545454u;
    if constexpr (ENC == QMM_Q5_K || ENC == QMM_Q6_K) asm volatile("" : "+v"(m_low), "+v"(c54));
    const ks_float4 zero4 = {0.f, 0.f, 0.f, 0.f};

    for (int c0 = 0; c0 < my_items; c0 += chunk) {
        const int ct = min(chunk, my_items - c0);
        for (int g = g_first; g < g_end; g++) {
            const int sb = g * waves + wave;
            float expert_weight = 1.0f;
            bool counts = true;
            if constexpr (EX == kSmallOverExperts) {
                const int of = min(sb / row_blocks, ex.r.top - 1);
                counts = __builtin_amdgcn_readlane(token_ids, of) >= 0;
                expert_weight = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, token_weights), of));
            }
            if (sb < nblk) {  // (all wavefronts but for the last group)
            if (groups > 1 && c0 + g > g_first) {
                xraw_t xr[MROWS];
#pragma unroll
                for (int j = 0; j < MROWS; j++) xr[j] = *(const xraw_t*)((const uint8_t*)lhs_at(j, sb) + a_lane);
                if constexpr (PART) leave_out(xr, sb);
                narrow(xr, ring + (slot ^ 1) * kSlot);
            }
            for (int t = 0; t < ct; t++) {
                // the next item: of the chunk, of the next group, of the next chunk
                int ng = g, nt = c0 + t + 1;
                if (t + 1 == ct) {
                    ng = g + 1, nt = c0;
                    if (ng == g_end || sb + waves >= nblk) ng = g_first, nt = c0 + ct;
                }
                if (nt < my_items) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (what was read from that slot is in registers)
                    issue(ng * waves + wave, nt, slot ^ 1);
                    wait_vmcnt<kLoads>();
                } else {
                    wait_vmcnt<0>();
                }
                const uint8_t* const lb = ring + slot * kSlot + nn * I::kRow;
                float v[LR];
                if constexpr (kQ8) {
                    // codes less 8, times 16, as signed bytes: the dot products of a block come out exact; v = sum of dot / 16 * (d_w d_a), the product of two fp16 numbers exact in fp32
                    const uint32_t* const l32 = (const uint32_t*)lb;
                    float u[2][LR];  // two chains of sums
#pragma unroll
                    for (int j = 0; j < LR; j++) u[0][j] = u[1][j] = 0.0f;
                    // PART: the row begins 0 or 2 bytes into its pieces; behind the last of them, its four bytes more
                    const uint32_t skew = PART ? ((uint32_t)(nn % kTile) * row_bytes + window(sb % row_blocks)) & 2u : 0u;
                    const uint32_t behind = PART ? ((const uint32_t*)(ring + slot * kSlot + I::kSlot))[nn] : 0u;
#pragma unroll
                    for (int b = 0; b < 8; b++) {
                        const int at = (18 * b + 2) >> 2;
                        uint32_t x;  // the block begins at 0 or 2 mod 4
                        if constexpr (PART) {
                            const uint32_t* const p = l32 + (18 * b >> 2) + (b & 1) + kg + (b & 1 ? 0u : skew >> 1);
                            x = __builtin_amdgcn_alignbyte(b == 7 && kg == 3 ? behind : p[1], p[0], b & 1 ? skew : skew ^ 2u);
                        } else if ((18 * b + 2) % 4 == 0) x = l32[at + kg];
                        else x = __builtin_amdgcn_alignbyte(l32[at + kg + 1], l32[at + kg], 2);
                        const half2v dp = __builtin_bit_cast(half2v, l32[(18 * b) >> 2]);
                        const _Float16 dw = PART ? __builtin_bit_cast(_Float16, *(const uint16_t*)(lb + 18 * b + skew)) : (18 * b) % 4 ? dp.y : dp.x;
                        const u32x2 w = {((x << 4) & 0xF0F0F0F0u) ^ 0x80808080u, (x & 0xF0F0F0F0u) ^ 0x80808080u};
                        const ks_int4 dot = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, fc[b]), __builtin_bit_cast(long, w), ks_int4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                        for (int j = 0; j < LR; j++) {
                            const uint32_t pair = fd[j][b >> 1];  // (a bit cast of the element itself takes the first one)
                            const half2v da2 = __builtin_bit_cast(half2v, pair);
                            u[b & 1][j] = fmaf((float)dot[j], fmaf((float)dw, (float)(b & 1 ? da2.y : da2.x), 0.0f), u[b & 1][j]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < LR; j++) v[j] = 0.0625f * (u[0][j] + u[1][j]);
                } else if constexpr (ENC == QMM_Q6_K) {
                    const uint32_t* const l32 = (const uint32_t*)lb;
                    const uint32_t skew = 2u * (((uint32_t)nn * (uint32_t)row_blocks + (uint32_t)(EX == kSmallOverExperts ? sb % row_blocks : sb)) & 1u);  // (16 rows of a tile: n0 is even)
                    auto rd = [&](int dw) __attribute__((always_inline)) { return __builtin_amdgcn_alignbyte(l32[dw + 1], l32[dw], skew); };
                    const uint4 s4 = *(const uint4*)(lb + 192);
                    const uint32_t tail = l32[55];  // bytes 208 .. 211
                    const uint32_t sd[4] = {__builtin_amdgcn_alignbyte(s4.y, s4.x, skew), __builtin_amdgcn_alignbyte(s4.z, s4.y, skew),
                                            __builtin_amdgcn_alignbyte(s4.w, s4.z, skew), __builtin_amdgcn_alignbyte(tail, s4.w, skew)};
                    const float d = h2f((uint16_t)(tail >> (8 * skew)));
                    const ks_half4 off96 = {(_Float16)96.0f, (_Float16)96.0f, (_Float16)96.0f, (_Float16)96.0f};
                    float u[2][RN];  // two chains of sums
#pragma unroll
                    for (int r = 0; r < RN; r++) u[0][r] = u[1][r] = 0.0f;
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int e2 = 0; e2 < 2; e2++) {
                            if constexpr (RN == 4) __builtin_amdgcn_sched_barrier(0);  // (with more results on their way at once the compiler spills)
                            const uint32_t QH = rd(32 + 8 * h + 4 * e2 + kg);
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                const int gr = 8 * h + 2 * c + e2;  // scale group: weights 128 h + 32 c + 16 e2 + (0..15)
                                const uint32_t QL = rd(16 * h + 8 * (c & 1) + 4 * e2 + kg);
                                const uint32_t lo = (c >> 1) ? QL & 0xF0F0F0F0u : (QL << 4) & 0xF0F0F0F0u;
                                const uint32_t hi = ((QH >> (2 * c)) & m_low) | c54;
                                const uint2 bq = make_uint2(__builtin_amdgcn_perm(hi, lo, 0x05010400u), __builtin_amdgcn_perm(hi, lo, 0x07030602u));
                                const ks_half4 bw = __builtin_bit_cast(ks_half4, bq) - off96;
                                const float cs = (float)((int)(sd[gr >> 2] << (24 - 8 * (gr & 3))) >> 24);
                                const ks_float4 P = __builtin_amdgcn_mfma_f32_16x16x16f16(fq[gr], bw, zero4, 0, 0, 0);
#pragma unroll
                                for (int r = 0; r < RN; r++) u[h][r] = fmaf(cs, P[r], u[h][r]);
                            }
                        }
#pragma unroll
                    for (int j = 0; j < LR; j++) v[j] = d * (PL == 2 ? (u[0][PL * j] + u[1][PL * j]) + (u[0][PL * j + PL - 1] + u[1][PL * j + PL - 1]) : u[0][j] + u[1][j]);
                } else {
                    const uint4 hdr = *(const uint4*)lb;
                    constexpr int kQs = ENC == QMM_Q4_K ? 16 : 48;
                    const uint4 q0 = *(const uint4*)(lb + kQs + 32 * kg), q1 = *(const uint4*)(lb + kQs + 16 + 32 * kg);
                    // 6-bit scales and mins of sub-blocks 2 kg, 2 kg + 1 (4 .. 7 use the split encoding)
                    const int sh = 16 * (kg & 1);
                    const uint32_t p0 = (hdr.y >> sh) & 0xffffu, p1 = (hdr.z >> sh) & 0xffffu, p2 = (hdr.w >> sh) & 0xffffu;
                    const uint32_t sc_pair = kg >= 2 ? ((p2 & 0x0F0Fu) | ((p0 >> 2) & 0x3030u)) : (p0 & 0x3F3Fu);
                    const uint32_t mn_pair = kg >= 2 ? (((p2 >> 4) & 0x0F0Fu) | ((p1 >> 2) & 0x3030u)) : (p1 & 0x3F3Fu);
                    float d = h2f((uint16_t)(hdr.x & 0xffffu));
                    // what the codes around their middle leave out: (mid d sc - dmin mn) times the sums of the lhs, both as two fp16 terms, the former times a power of two that
                    // brings the largest it can be below 2^15
                    constexpr float kMid = ENC == QMM_Q4_K ? 8.0f : 16.0f;
                    const float dm = kMid * d, dmin = h2f((uint16_t)(hdr.x >> 16)), e0 = (float)(sc_pair & 0xffu), e1 = (float)(sc_pair >> 8);
                    const int scale = 15 - __builtin_amdgcn_frexp_expf(63.0f * (fabsf(dm) + fabsf(dmin)));
                    const float o0 = __builtin_amdgcn_ldexpf(fmaf(dm, e0, -(dmin * (float)(mn_pair & 0xffu))), scale), o1 = __builtin_amdgcn_ldexpf(fmaf(dm, e1, -(dmin * (float)(mn_pair >> 8))), scale);
                    const half2v oh = to_half2(o0, o1), ol = to_half2(fmaf((float)oh.x, -1.0f, o0), fmaf((float)oh.y, -1.0f, o1));
                    const uint32_t ohb = __builtin_bit_cast(uint32_t, oh), olb = __builtin_bit_cast(uint32_t, ol);
                    const half8 offs = pack4(__builtin_amdgcn_perm(ohb, ohb, 0x01000100u), (olb & 0xffffu) | (ohb & 0xffff0000u), (ohb >> 16) | (olb & 0xffff0000u), 0u);
                    const uint32_t qd[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
                    ks_float4 P = zero4, Q = zero4;  // two chains: low and high nibbles
                    if constexpr (ENC == QMM_Q4_K) {
                        const uint32_t M1 = 0x000F000Fu, M2 = 0x00F000F0u;
                        // 64 sc for the low nibbles (q * 2^-24), 4 sc for the high ones (16 q * 2^-24): the operand is sc * (q - 8) * 2^-18 (as sc * q * 2^-24, always a subnormal, the matrix core
                        // drops low bits of the products)
                        const uint32_t sp_lo = to_half2_bits(64.0f * e0, 64.0f * e0), sp_hi = to_half2_bits(4.0f * e1, 4.0f * e1);
                        const uint32_t np_lo = pk_mul(sp_lo, 0x80088008u), np_hi = pk_mul(sp_hi, 0x80808080u);  // -8 * 2^-24, -128 * 2^-24 times it
                        d *= 262144.0f;
#pragma unroll
                        for (int p = 0; p < 4; p++) {
                            const uint32_t x0 = qd[2 * p], x1 = qd[2 * p + 1], y0 = x0 >> 8, y1 = x1 >> 8;
                            const half8 blo = pack4(pk_fma(x0 & M1, sp_lo, np_lo), pk_fma(y0 & M1, sp_lo, np_lo), pk_fma(x1 & M1, sp_lo, np_lo), pk_fma(y1 & M1, sp_lo, np_lo));
                            const half8 bhi = pack4(pk_fma(x0 & M2, sp_hi, np_hi), pk_fma(y0 & M2, sp_hi, np_hi), pk_fma(x1 & M2, sp_hi, np_hi), pk_fma(y1 & M2, sp_hi, np_hi));
                            P = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[p][0], blo, P, 0, 0, 0);
                            Q = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[p][1], bhi, Q, 0, 0, 0);
                        }
                    } else {
                        const uint4 h0 = *(const uint4*)(lb + 16), h1 = *(const uint4*)(lb + 32);  // fifth bits: bit j of byte i, column i of sub-block j
                        const uint32_t hd[8] = {h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w};
                        const uint32_t s_lo = to_half2_bits(e0, e0), s_hi = to_half2_bits(e1, e1), n_lo = to_half2_bits(-80.0f * e0, -80.0f * e0), n_hi = to_half2_bits(-80.0f * e1, -80.0f * e1);
#pragma unroll
                        for (int p = 0; p < 4; p++) {
                            uint32_t lo[4], hi[4];
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const uint32_t x = qd[2 * p + i], f = hd[2 * p + i] >> (2 * kg);
                                const uint32_t xl = (x << 4) & 0xF0F0F0F0u, xh = x & 0xF0F0F0F0u, fl = (f & m_low) | c54, fh = ((f >> 1) & m_low) | c54;
                                lo[2 * i] = pk_fma(__builtin_amdgcn_perm(fl, xl, 0x05010400u), s_lo, n_lo);
                                lo[2 * i + 1] = pk_fma(__builtin_amdgcn_perm(fl, xl, 0x07030602u), s_lo, n_lo);
                                hi[2 * i] = pk_fma(__builtin_amdgcn_perm(fh, xh, 0x05010400u), s_hi, n_hi);
                                hi[2 * i + 1] = pk_fma(__builtin_amdgcn_perm(fh, xh, 0x07030602u), s_hi, n_hi);
                            }
                            P = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[p][0], pack4(lo[0], lo[1], lo[2], lo[3]), P, 0, 0, 0);
                            Q = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[p][1], pack4(hi[0], hi[1], hi[2], hi[3]), Q, 0, 0, 0);
                        }
                    }
                    const ks_float4 O = __builtin_amdgcn_mfma_f32_16x16x32_f16(fs, offs, zero4, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < LR; j++) {
                        float sum = P[PL * j] + Q[PL * j], off = O[PL * j];
                        if constexpr (PL == 2) sum += P[PL * j + PL - 1] + Q[PL * j + PL - 1], off += O[PL * j + PL - 1];
                        v[j] = fmaf(d, sum, __builtin_amdgcn_ldexpf(off, -scale));
                    }
                }
                float* const mine = accs + ((t * waves + wave) * LR) * 64 + lane;
#pragma unroll
                for (int j = 0; j < LR; j++) {
                    float y = kQ8 ? v[j] : bs[j] * v[j];
                    if constexpr (EX == kSmallOverExperts) y = counts ? expert_weight * y : 0.0f;
                    mine[j * 64] = y;
                }
                slot ^= 1;
            }
            }
            __syncthreads();
            // the group's result (matrix row 16 tile + nn, lhs row kg + 4 j): dealt to the wavefronts, which add it to that of the groups before
            const int live = min(waves, nblk - g * waves);
            for (int q = wave; q < ct / kEach * LR; q += waves) {
                const int t = q / LR * kEach, j = q % LR, row = row0 + kg + 4 * j;
                float s[kEach];
#pragma unroll
                for (int h = 0; h < kEach; h++) {
                    const float* const src = accs + (((t + h) * waves) * LR + j) * 64 + lane;
                    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    int w = 0;
                    for (; w + 4 <= live; w += 4)
#pragma unroll
                        for (int i = 0; i < 4; i++) c[i] += src[(w + i) * LR * 64];
#pragma unroll
                    for (int i = 0; i < 3; i++)
                        if (w + i < live) c[i] += src[(w + i) * LR * 64];
                    s[h] = (c[0] + c[1]) + (c[2] + c[3]);
                    if (groups > 1) {
                        float* const total = totals + ((t + h) * LR + j) * 64 + lane;
                        if (g > g_first) s[h] = *total + s[h];
                        if (g + 1 < g_end) *total = s[h];
                    }
                }
                if (g + 1 < g_end) continue;
                int n0, n;
                const int mat = matrix_of(c0 + t, n0, n);
                float r = s[0];
                if constexpr (MODE == kSmallGated) r = r / (1.0f + expf(-r)) * dpp_move<0x128>(r);  // (lanes nn < 8: gate, times up eight lanes on)
                if constexpr (MODE == kSmallPairs) r = r / (1.0f + expf(-r)) * s[kEach - 1];
                int64_t at = (int64_t)row * n + n0 + nn;
                if constexpr (EX == kSmallByExpert) {
                    if (row >= m) continue;
                    int pair = my_pairs[0];  // (j is no constant here)
#pragma unroll
                    for (int i = 1; i < LR; i++) pair = j == i ? my_pairs[i] : pair;
                    if (pair < 0) continue;
                    at = (int64_t)pair * n + n0 + nn;
                }
                if constexpr (EX == kSmallOverExperts) {
                    at = (int64_t)blockIdx.y * n + n0 + nn;
                    if (ex.residual && row < m && n0 + nn < n) r += ex.residual_bf16 ? load_f32((const uint16_t*)ex.residual, at) : load_f32((const float*)ex.residual, at);
                }
                if (row < m && nn < kTile && n0 + nn < n) {
                    if (out_bf16) ((uint16_t*)mats.out[mat])[at] = f2bf(r);
                    else mats.out[mat][at + (int64_t)part * m * n] = r;
                }
            }
            if (g + 1 < g_end || c0 + chunk < my_items) __syncthreads();
        }
    }
}

}  // namespace qmm
