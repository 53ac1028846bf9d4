// The experts' products on the matrix cores: weights packed as they lie in memory, unpacked between the matrix-core instructions, lhs rows gathered by the expert's list.
//
// One launch narrows every lhs row to fp16 once (a row's pieces in operand order, next to each other: [K / 32][fp32: hi, residual][4 pieces of 8 columns]); what an expert gets is picked by address, so a
// token's row is not copied to each of its experts.  Then a workgroup of four wavefronts takes up to 32 FM rows of one expert's run x 128 columns (gated: 64 of gate and the same 64 of up, whose
// results meet in LDS): each wavefront unpacks the weights of its 32 columns, the lhs goes global -> LDS directly, a chunk of 32 columns at a time into three or four buffers that all share.  A load brings
// 16 rows x 64 bytes, as memory has them; which of a row's pieces a lane asks for is turned by the row, so that the operands (piece p of 32 rows) are read back without bank conflicts.
// LDS is sized for two workgroups on a compute unit: an expert's K is short (8 units of 256 here and there), and what surrounds the products (finding the rows, the way to the first loads, the results) is
// hidden by the other one.  One workgroup of eight wavefronts x 256 columns instead: 2000 tokens, 8 of 64 experts, 1024 x 2048, Q4_K gate and up 205 us; matrix cores busy a third of the time.
//
// What bounds it: that case 187 us now (718 TFLOP/s), matrix cores busy 0.45 of it, vector units 0.53, two wavefronts a SIMD hide little of one behind the other; 9 % of the matrix instructions are for rows that are not
// there, and some compute units have nothing left for the last 15 %.  256 rows for each of the 64: 806 TFLOP/s, what the dense staged GEMM reaches on 16384 rows.  Q6_K down 500 fp32 rows, four products a weight: 99 us,
// matrix cores 0.47.  Q4_0 1408 x 2080, 301 rows, 4 of 16: 31 us, nine units of K one after the other, vector units 0.52.
//
// The grid counts groups of rows as if every expert's last one were a group more: how many rows an expert has is known on the device only.  A workgroup looks for its group in the offsets
// (a scan by one wavefront's lanes) and leaves if there is none; a group with few rows runs the body for as many.
//
// Arithmetic as in gemm_staged.hip: exact products of integer codes and fp16 values, fp32 sums, scales applied to the sums of a scale block.
#include <algorithm>
#include <type_traits>

#include "experts.h"
#include "staged_weights.h"

namespace qmm {

namespace {

struct EgArgs {
    const uint8_t* a16;    // [lhs rows][k / 32 rounded up to whole units][hi, fp32: residual] of 64 bytes
    const uint8_t* sums;   // [lhs rows][units][32 bytes]: sums of 32 columns, eight hi and eight lo parts; Q4_0: eight block scales, zeros
    const float* inv;      // [lhs rows]
    const uint8_t* w[2];
    int64_t stride[2];
    int lhs_top, n, k, units, gated;
    void* out;
    int out_bf16;
};

// The weights of one wavefront: loads to LDS, a unit ahead.
template <int ENC, bool CENTER>
struct EgStaged : StagedOf<ENC, 16, CENTER> {
    using Base = StagedOf<ENC, 16, CENTER>;
    static constexpr bool kQ8 = false;
    static constexpr int kBufs = 2, kAhead = Base::kLoads;
    __device__ __forceinline__ bool load_last(int) { return false; }
};
// Q4_0: a row's eight blocks of a unit from the last multiple of four on, in nine pieces of 16 bytes and four bytes that only rows which begin two bytes later need.  The fields of a row lie `skew` (0 or 2)
// bytes into its pieces.  Rows of any number of blocks: the unit that ends the row, where it is a partial one, is the first to be multiplied, comes through registers, and is zeros behind the row's end.  So the
// loads to LDS never read beyond a row: a row with skew has an odd number of blocks and ends in a partial unit (or the matrices do not begin at multiples of four, see experts_gemm_supported).
// Decoding as in Q40Weights: lane half g takes bytes 8 g .. 8 g + 7 of a block, low nibbles first.
struct EgQ40 : NoOffsets {
    static constexpr bool kQ8 = true, kMin = false;
    static constexpr int kPlanes = 1, kBufs = 2, kUnit = 8 * Q4_0_BPB, kPieces = kUnit / 16, kTotal = 32 * kPieces, kWide = (kTotal + 63) / 64, kLoads = kWide + 1, kAhead = kLoads;
    static constexpr int kTail = kTotal * 16, kStage = kTail + 128;
    const uint8_t* w;
    uint8_t* stage;
    const uint8_t* cur;
    const uint8_t* tail;
    uint32_t stage_lds, off[kWide], off_tail, skew, mine;  // mine: where the lane's row (of 32) begins
    int row_bytes, g, lane_;
    uint32_t x[2][3];
    uint32_t d[8], last;  // (of lanes g = 0; zero in the others)
    uint32_t top0 = code_top(0x64006400u), top1 = code_top(0x54005400u);
    struct __attribute__((packed, aligned(2))) Bytes16 {
        gd_u4 v;
    };
    // from w on
    __device__ __forceinline__ uint32_t row_at(const WeightTensors& t, int row) const { return (uint32_t)min(row, t.n - 1) * (uint32_t)row_bytes + ((uint32_t)(uintptr_t)t.w & 2u); }
    __device__ __forceinline__ void init(const WeightTensors& t, int n0, int lane, uint8_t* at) {
        g = lane >> 5;
        lane_ = lane;
        stage = at;
        stage_lds = lds_address(at);
        w = t.w - ((uintptr_t)t.w & 2);
        row_bytes = t.k / 32 * Q4_0_BPB;
        d[7] = 0;
        const int step = row_bytes < kUnit ? 0 : 16;  // (the only unit is partial: what is asked for in advance and never looked at stays within the row)
#pragma unroll
        for (int j = 0; j < kWide; j++) {
            const int i = min(j * 64 + lane, kTotal - 1), row = i / kPieces;
            off[j] = (row_at(t, n0 + row) & ~2u) + step * (i - row * kPieces);
        }
        mine = row_at(t, n0 + (lane & 31));
        skew = mine & 2u;
        off_tail = (mine & ~2u) + (skew && step ? kUnit : 0);
    }
    template <int J>
    __device__ __forceinline__ void issue(int unit, int buf) {
        const uint8_t* b = w + (int64_t)unit * kUnit;
        const uint32_t to = stage_lds + buf * kStage;
        if constexpr (J < kWide) {
            if (J * 64 + 63 < kTotal || J * 64 + lane_ < kTotal) load16_to_lds(off[J], b, to + J * 1024);
        } else if (lane_ < 32) {
            load4_to_lds(b + off_tail, to + kTail);
        }
    }
    // the partial unit at the rows' end, to the first buffer
    __device__ __forceinline__ bool load_last(int unit) {
        const int left = row_bytes - unit * kUnit;
        if (left == kUnit) return false;
#pragma unroll
        for (int j = 0; j < kWide; j++) {
            const int i = min(j * 64 + lane_, kTotal - 1), row = i / kPieces, piece = 16 * (i - row * kPieces);
            const uint32_t begin = (uint32_t)__shfl((int)mine, row);
            // the last 16 bytes of the row, moved down to the place the piece would have (rows are at least 18 bytes long)
            const int over = max(piece + 16 - left - (int)(begin & 2u), 0);
            const gd_u4 v = ((const Bytes16*)(w + (int64_t)unit * kUnit + (begin & ~2u) + piece - over))->v;
            uint64_t lo = v.x | (uint64_t)v.y << 32, hi = v.z | (uint64_t)v.w << 32;
            if (over >= 16) lo = hi = 0;
            else if (over >= 8) { lo = hi >> (8 * over - 64); hi = 0; }
            else if (over > 0) { lo = (lo >> (8 * over)) | (hi << (64 - 8 * over)); hi >>= 8 * over; }
            if (j * 64 + 63 < kTotal || j * 64 + lane_ < kTotal) *(gd_u4*)(stage + j * 1024 + lane_ * 16) = gd_u4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
        }
        return true;
    }
    // Block b begins with its scale at 18 b + skew of the row; the lane's eight code bytes are two bytes and 8 g further: from a multiple of four on, or two bytes behind one.
    template <int B>
    __device__ __forceinline__ void read_block() {
        const uint32_t* const p = (const uint32_t*)(cur + 8 * g + (B & 1 ? 18 * B + 2 : 18 * B + 2 * skew));
        x[B & 1][0] = p[0];
        x[B & 1][1] = p[1];
        x[B & 1][2] = B == 7 ? *(const uint32_t*)tail : p[2];
    }
    __device__ __forceinline__ void open(int, int buf) {
        const uint8_t* const b = stage + buf * kStage;
        cur = b + (lane_ & 31) * kUnit;
        tail = g ? b + kTail + 4 * (lane_ & 31) : cur + 136;
        read_block<0>();
        last = d[7];  // (the last block is scaled in the next unit)
#pragma unroll
        for (int i = 0; i < 8; i++) d[i] = g ? 0u : (uint32_t)*(const uint16_t*)(cur + skew + 18 * i);
    }
    template <int T>
    __device__ __forceinline__ void step(int, half8 (&b)[1]) const {
        constexpr int blk = T >> 1;
        const uint32_t turn = blk & 1 ? skew : skew ^ 2u;
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t q = __builtin_amdgcn_alignbyte(x[blk & 1][i + 1], x[blk & 1][i], turn), y = q >> 8;
            if constexpr ((T & 1) == 0) {
                v[2 * i] = pk_add((q & 0x000F000Fu) | top0, 0xE408E408u);  // 1024 + q - 1032
                v[2 * i + 1] = pk_add((y & 0x000F000Fu) | top0, 0xE408E408u);
            } else {
                v[2 * i] = pk_add((q & 0x00F000F0u) | top1, 0xD480D480u);  // 64 + q - 72
                v[2 * i + 1] = pk_add((y & 0x00F000F0u) | top1, 0xD480D480u);
            }
        }
        b[0] = pack4(v[0], v[1], v[2], v[3]);
    }
    template <int T>
    __device__ __forceinline__ void before_step() {
        if constexpr ((T & 1) == 0 && T < 14) read_block<(T >> 1) + 1>();
    }
    template <int B>
    __device__ __forceinline__ half8 scale_operand(int) const {
        const uint32_t v = (B == 7 ? last : d[B]) << (16 * (B & 1));
        return pack4(B >> 1 == 0 ? v : 0u, B >> 1 == 1 ? v : 0u, B >> 1 == 2 ? v : 0u, B >> 1 == 3 ? v : 0u);
    }
};
template <int ENC, bool CENTER>
using EgWeights = std::conditional_t<ENC == QMM_Q4_0, EgQ40, EgStaged<ENC == QMM_Q4_0 ? QMM_Q4_K : ENC, CENTER>>;

constexpr int kEgWaves = 4;
// Steps of 16 columns in a chunk: a barrier for each chunk.
constexpr int eg_steps(int enc) { return enc == QMM_Q4_K || enc == QMM_Q4_0 ? 4 : 2; }
struct EgRow {
    int64_t at;  // of the row's results, in values; -1: none
    float inv;
    int pad;
};
// Rows of a workgroup at most, in 32s: what the registers and half a compute unit's LDS hold.
constexpr int eg_most(int enc, bool hilo) { return hilo || enc == QMM_Q4_0 ? 2 : 4; }
template <int ENC, int FM, bool HILO>
struct EgLds {
    using W = EgWeights<ENC, HILO>;
    static constexpr int kPer = HILO ? 2 : 1, kSteps = eg_steps(ENC), kChunk = FM * 1024 * kSteps * kPer, kWeights = kEgWaves * W::kBufs * W::kStage, kSums = W::kMin || W::kQ8 ? 2 * FM * 1024 : 0;
    static constexpr int kResultRow = 40, kResults = kEgWaves * 32 * std::min(FM, 2) * kResultRow * 4, kInfoBytes = 32 * FM * (int)sizeof(EgRow);
    static constexpr int bytes(int bufs) { return std::max(bufs * kChunk + kWeights + kSums, kResults) + kInfoBytes; }
    static constexpr int kShare = kLdsPerCu / (FM == 1 && bytes(2) <= kLdsPerCu / 3 ? 3 : 2);
    static constexpr int kBufs = bytes(4) <= kShare ? 4 : bytes(3) <= kShare ? 3 : 2;
    static constexpr int kW = kBufs * kChunk, kS = kW + kWeights, kInfo = std::max(kS + kSums, kResults), kBytes = bytes(kBufs);
    static_assert(kBytes <= kLdsPerCu / 2, "two on a compute unit");
};

__device__ __forceinline__ float silu(float v) {
    // v / (1 + exp(-v)): the product v L as two terms, so that the exponential is right to the last bits for any v
    const float p = v * -1.44269504088896f, rest = fmaf(v, -1.44269504088896f, -p), e = __builtin_amdgcn_exp2f(p);
    return v * __builtin_amdgcn_rcpf(1.0f + fmaf(e, rest * 0.693147180559945f, e));
}

template <int ENC, int FM, bool HILO, bool GATED>
__device__ __forceinline__ void experts_tile(const EgArgs& p, const Routing& r, const ExpertRows& rows, int col_tile) {
    using W = EgWeights<ENC, HILO>;
    using L = EgLds<ENC, FM, HILO>;
    constexpr int kPer = L::kPer, kBufs = L::kBufs, kSteps = L::kSteps, kChunks = 16 / kSteps, kTotal = FM * kSteps * kPer, kLoads = (kTotal + kEgWaves - 1) / kEgWaves;  // loads of a chunk, of a wavefront
    constexpr bool kHasSums = W::kMin || W::kQ8, kUnit = W::kQ8 || (W::kMin && HILO);                   // kUnit: a unit's sums apart from the running ones
    constexpr int kAhead = W::kAhead + (kHasSums ? 1 : 0);
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), row = lane & 31, g = lane >> 5;
    constexpr int kCols = GATED ? 64 : 128;
    const int mat = GATED ? wave >> 1 : 0, n0 = col_tile * kCols + 32 * (GATED ? wave & 1 : wave);
    EgRow* const info = (EgRow*)(smem + L::kInfo);
    WeightTensors wt{p.w[mat] + rows.expert * p.stride[mat], nullptr, nullptr, p.n, p.k, 0};
    const int units = p.units, last_chunk = units * kChunks - 1;
    auto unit_at = [&](int u) __attribute__((always_inline)) { return !W::kQ8 ? u : u == 0 ? units - 1 : u - 1; };  // Q4_0: the last unit first
    const uint32_t lds0 = lds_address(smem);
    W w;
    w.init(wt, n0, lane, smem + L::kW + wave * W::kBufs * W::kStage);
    auto issue_weights = [&](int unit, int buf) __attribute__((always_inline)) {
        unrolled<W::kAhead>([&](auto j) __attribute__((always_inline)) { w.template issue<decltype(j)::value>(unit, buf); });
    };
    auto lhs_row = [&](int i) __attribute__((always_inline)) { return max(pair_at(r, rows.first + min(i, rows.count - 1)), 0) / p.lhs_top; };
    // a row of a chunk is kPieces of 16 bytes; a piece's place is turned by the row, so that the same piece of 16 rows lies in all banks
    constexpr int kPieces = 2 * kSteps, kRows = 64 / kPieces;  // rows of a load
    auto turned = [&](int piece, int of_row) __attribute__((always_inline)) { return piece ^ ((of_row * kPieces >> 4) & (kPieces - 1)); };
    // this wavefront's loads of a chunk: number first + j of them, kRows rows each
    const int first = min(wave * kLoads, kTotal - kLoads);
    const uint8_t* src[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
        const int i = first + j, plane = i / (FM * kSteps), at_row = i % (FM * kSteps) * kRows + lane / kPieces;
        src[j] = p.a16 + (int64_t)lhs_row(at_row) * units * (512 * kPer) + plane * (32 * kSteps) + turned(lane % kPieces, at_row) * 16;
    }
    const uint8_t* sums_src = nullptr;
    const int sums_tile = wave % FM;
    if constexpr (kHasSums) sums_src = p.sums + (int64_t)lhs_row(32 * sums_tile + row) * units * 32 + g * 16;
    int info_row = 0;
    if (threadIdx.x < 32 * FM) {
        const int pair = pair_at(r, rows.first + min((int)threadIdx.x, rows.count - 1));
        info_row = max(pair, 0) / p.lhs_top;
        info[threadIdx.x].at = (int)threadIdx.x < rows.count && pair >= 0 ? (int64_t)pair * p.n : -1;
    }
    auto issue_lhs = [&](int chunk, int buf) __attribute__((always_inline)) {
        const int c = min(chunk, last_chunk);
        const int64_t at = (int64_t)(!W::kQ8 ? c : c < kChunks ? c + last_chunk + 1 - kChunks : c - kChunks) * (32 * kSteps * kPer);
#pragma unroll
        for (int j = 0; j < kLoads; j++) load16_to_lds(src[j] + at, (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + buf * L::kChunk + (first + j) * 1024)));
    };
    auto issue_sums = [&](int unit, int buf) __attribute__((always_inline)) {
        if constexpr (kHasSums) load16_to_lds(sums_src + (int64_t)unit * 32, (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + L::kS + (buf * FM + sums_tile) * 1024)));
    };

    float16v T[FM], P[FM], M, U[kUnit ? FM : 1], B[2][FM], S[FM];  // Q4_0: products of two blocks, scales
    half8 scales[FM];
#pragma unroll
    for (int a = 0; a < FM; a++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            T[a][i] = P[a][i] = B[1][a][i] = 0.0f;
            scales[a][i & 7] = 0;
            if constexpr (kUnit) U[a][i] = 0.0f;
        }
    const float16v zero16 = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    // where a lane's operands of the steps of a chunk lie
    uint32_t at_step[kSteps];
#pragma unroll
    for (int t = 0; t < kSteps; t++) at_step[t] = row * (32 * kSteps) + turned(2 * t + g, row) * 16;
    half8 af[2][FM][kPer], b[2][W::kPlanes];
    auto read_lhs = [&](int step, int slot, uint32_t base) __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < FM; a++)
#pragma unroll
            for (int q = 0; q < kPer; q++) af[slot][a][q] = *(const half8*)(smem + base + at_step[step] + (q * FM + a) * (1024 * kSteps));
    };

    // (From here on the loads are counted: an ordinary one among them would wait for all.)
    if (!w.load_last(unit_at(0))) issue_weights(unit_at(0), 0);
    issue_sums(unit_at(0), 0);
#pragma unroll
    for (int c = 0; c < kBufs - 1; c++) issue_lhs(c, c);
    wait_vmcnt<(kBufs - 2) * kLoads>();
    __syncthreads();
    issue_lhs(kBufs - 1, kBufs - 1);
    w.open(unit_at(0), 0);
    read_lhs(0, 0, 0);
    w.template step<0>(0, b[0]);
    float d = 0.0f;
    int buf = 0;  // of the current chunk
    for (int u = 0; u < units; u++) {
        const int next = unit_at(min(u + 1, units - 1));
        // (nobody reads the sums and weights of the unit before any more)
        issue_weights(next, (u + 1) & 1);
        issue_sums(next, (u + 1) & 1);
        float dmin = 0.0f, dnext = 0.0f;
        if constexpr (!W::kQ8) {
            dnext = w.scale(0);
            if constexpr (W::kMin && !HILO) dmin = w.min_scale(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        unrolled<16>([&](auto tt) __attribute__((always_inline)) {
            constexpr int t = decltype(tt)::value, cur = t & 1, entered = t / kSteps + 1;
            if constexpr (t % kSteps == kSteps - 1) {
                // The next chunk has arrived (asked for kBufs - 1 boundaries ago; younger: the chunks after it, and the next unit's weights and sums where they were asked for since), and every wavefront has
                // read this one's operands into registers: its buffer takes the chunk after those that are there.  At a unit's end the weights are older than the chunk.
                static_assert(kBufs - 1 < kChunks, "the weights of the next unit are older than its first chunk");
                wait_vmcnt<(kBufs - 2) * kLoads + (entered <= kBufs - 1 ? kAhead : 0)>();
                __syncthreads();
                issue_lhs(u * kChunks + entered + kBufs - 1, buf);
                buf = buf == kBufs - 1 ? 0 : buf + 1;
            }
            read_lhs((t + 1) % kSteps, cur ^ 1, (uint32_t)(buf * L::kChunk));
            if constexpr (t + 1 == 16) w.open(next, (u + 1) & 1);
            w.template before_step<t>();
            // one row tile every three steps, the last at steps 14 and 15
            constexpr int min_a = (t - 14 + 3 * (FM - 1)) / 3, min_at = 14 - 3 * (FM - 1);
            constexpr bool min_now = W::kMin && t >= min_at && (t - min_at) % 3 == 0, min_add = W::kMin && t > min_at && (t - min_at) % 3 == 1;
            half8 sf;
            if constexpr (min_now) sf = *(const half8*)(smem + L::kS + ((u & 1) * FM + min_a) * 1024 + lane * 16);
            if constexpr (W::kMin && HILO && t < 5) {
                if constexpr (t == 0) dmin = w.open_offsets();
                else w.template add_offsets<t - 1>();
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (W::kQ8) {
// The products of a block are scaled while the next one's run.  Its scales as a matrix: the row's scale in slot b times the weight's in the same slot.
                constexpr int done = (t / 2 + 7) % 8, at = t / 2 % 2;
#pragma unroll
                for (int a = 0; a < FM; a++) {
                    B[at][a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[cur][a][0], b[cur][0], t % 2 ? B[at][a] : zero16, 0, 0, 0);
                    if constexpr (t % 2 == 0) S[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(scales[a], w.template scale_operand<done>(0), zero16, 0, 0, 0);
                }
                if constexpr (t % 2 == 1) {
#pragma unroll
                    for (int a = 0; a < FM; a++) {
#pragma unroll
                        for (int i = 0; i < 16; i++) U[a][i] = done == 0 ? B[at ^ 1][a][i] * S[a][i] : fmaf(B[at ^ 1][a][i], S[a][i], U[a][i]);
                        if constexpr (done == 7) {
#pragma unroll
                            for (int i = 0; i < 16; i++) T[a][i] += U[a][i];
                            asm volatile("" : "+v"(T[a]));
                        } else {
                            asm volatile("" : "+v"(U[a]));
                        }
                    }
                }
                if constexpr (t == 0) {
#pragma unroll
                    for (int a = 0; a < FM; a++) scales[a] = *(const half8*)(smem + L::kS + ((u & 1) * FM + a) * 1024 + lane * 16);
                }
            } else if constexpr (t == 0) {
#pragma unroll
                for (int a = 0; a < FM; a++) {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        if constexpr (kUnit) T[a][i] += fmaf(d, P[a][i], U[a][i]);
                        else T[a][i] = fmaf(d, P[a][i], T[a][i]);
                    }
                    asm volatile("" : "+v"(T[a]));
#pragma unroll
                    for (int pl = 0; pl < W::kPlanes; pl++)
#pragma unroll
                        for (int q = 0; q < kPer; q++) P[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[cur][a][q], b[cur][pl], q || pl ? P[a] : zero16, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
                d = dnext;
            } else {
#pragma unroll
                for (int pl = 0; pl < W::kPlanes; pl++)
#pragma unroll
                    for (int q = 0; q < kPer; q++)
#pragma unroll
                        for (int a = 0; a < FM; a++) P[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[cur][a][q], b[cur][pl], P[a], 0, 0, 0);
            }
            if constexpr (min_now) {
                if constexpr (HILO) {
                    M = __builtin_amdgcn_mfma_f32_32x32x16_f16(sf, w.offsets_lo(), zero16, 0, 0, 0);
                    M = __builtin_amdgcn_mfma_f32_32x32x16_f16(sf, w.offsets_hi(), M, 0, 0, 0);
                } else {
                    M = __builtin_amdgcn_mfma_f32_32x32x16_f16(sf, w.min_operand(0), zero16, 0, 0, 0);
                }
            }
            if constexpr (min_add) {  // (a step later: the product takes its time)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    if constexpr (kUnit) U[min_a][i] = dmin * M[i];
                    else T[min_a][i] = fmaf(dmin, M[i], T[min_a][i]);
                }
            }
            w.template step<(t + 1) % 16>(0, b[cur ^ 1]);
            if constexpr (W::kQ8 || t != 0) {
                constexpr int kMfma = FM * kPer * W::kPlanes * (W::kQ8 && t % 2 == 0 ? 2 : 1);
                constexpr int kValu = (W::kPlanes == 2 ? 28 : 12) + (min_add ? 16 : 0) + (W::kQ8 && t % 2 ? 16 * FM : 0);  // spread evenly
                unrolled<kMfma + (min_now ? (HILO ? 2 : 1) : 0)>([&](auto) __attribute__((always_inline)) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x2, (kValu + kMfma - 1) / kMfma, 0);
                });
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    }
    if constexpr (W::kQ8) {
#pragma unroll
        for (int a = 0; a < FM; a++) {
            S[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(scales[a], w.template scale_operand<7>(0), zero16, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 16; i++) T[a][i] += fmaf(B[1][a][i], S[a][i], U[a][i]);
        }
    } else {
#pragma unroll
        for (int a = 0; a < FM; a++)
#pragma unroll
            for (int i = 0; i < 16; i++) T[a][i] = kUnit ? T[a][i] + fmaf(d, P[a][i], U[a][i]) : fmaf(d, P[a][i], T[a][i]);
    }
    if (threadIdx.x < 32 * FM) info[threadIdx.x].inv = p.inv[info_row];
    wait_vmcnt<0>();
    __syncthreads();  // nothing is on its way into the buffers any more, which now take the results
    constexpr int kRow = L::kResultRow, kTiles = std::min(FM, 2), kTile = 32 * kTiles * kRow;
    static_assert(FM % kTiles == 0, "every turn has all its rows: beyond the last one `info` holds no place to store to");
    float* const mine = (float*)smem + wave * kTile;
#pragma unroll
    for (int a0 = 0; a0 < FM; a0 += kTiles) {
        if (a0) __syncthreads();
#pragma unroll
        for (int a = a0; a < FM && a < a0 + kTiles; a++)
#pragma unroll
            for (int i = 0; i < 16; i++) mine[(32 * (a - a0) + 8 * (i >> 2) + 4 * g + (i & 3)) * kRow + row] = T[a][i];
        __syncthreads();
        // two rows of 32 columns at a time; gated: the wavefronts of gate take the first half of the rows, those of up the second
        const int strip = GATED ? wave & 1 : wave, col = col_tile * kCols + 32 * strip + row;
        const float* const y = (const float*)smem + strip * kTile;
        constexpr int kMine = GATED ? 16 * kTiles : 32 * kTiles;
        const int from = GATED ? (wave >> 1) * kMine : 0;
        if (col < p.n) {
            for (int i0 = from + g; i0 < from + kMine; i0 += 8) {
                EgRow e[4];
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int i = i0 + 2 * j;
                    e[j] = info[32 * a0 + i];
                    v[j] = y[i * kRow + row] * e[j].inv;
                    if constexpr (GATED) v[j] = silu(v[j]) * (y[2 * kTile + i * kRow + row] * e[j].inv);
                }
                if (p.out_bf16) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (e[j].at >= 0) ((uint16_t*)p.out)[e[j].at + col] = f2bf(v[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (e[j].at >= 0) ((float*)p.out)[e[j].at + col] = v[j];
                }
            }
        }
    }
}

template <bool GATED>
__device__ __forceinline__ void zero_tile(const EgArgs& p, const Routing& r, const ExpertRows& rows, int col_tile) {
    constexpr int kCols = GATED ? 64 : 128;
    const int col = col_tile * kCols + (int)threadIdx.x % kCols;
    if (col >= p.n) return;
    for (int i = (int)threadIdx.x / kCols; i < rows.count; i += 64 * kEgWaves / kCols) {
        const int pair = pair_at(r, rows.first + i);
        if (pair < 0) continue;
        if (p.out_bf16) ((uint16_t*)p.out)[(int64_t)pair * p.n + col] = 0;
        else ((float*)p.out)[(int64_t)pair * p.n + col] = 0.0f;
    }
}

template <int ENC, int FM, bool HILO, bool GATED>
__global__ __launch_bounds__(64 * kEgWaves, 2) void experts_gemm_kernel(EgArgs p, Routing r) {
    // The tiles, those of one group of rows after the other, in eight equal parts: one for each XCD (ids congruent mod 8), in whose L2 an expert's weights and rows then are, once.
    const uint32_t cols = (uint32_t)(p.n + (GATED ? 63 : 127)) / (GATED ? 64 : 128);
    int col_tile = 0;
    const ExpertRows rows = uniform(find_rows_of<32 * FM>(r, threadIdx.x & 63, [&](int groups) {
        const int64_t tiles = (int64_t)groups * cols, place = (tiles * blockIdx.x >> 3) + blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
        if (place >= tiles * (blockIdx.x + 1) >> 3) return -1;
        const int group = (int)((uint32_t)place / cols);
        col_tile = __builtin_amdgcn_readfirstlane((int)((uint32_t)place - (uint32_t)group * cols));
        return group;
    }));
    if (rows.count == 0) return;
    if (rows.expert >= r.experts) return zero_tile<GATED>(p, r, rows, col_tile);
    if constexpr (FM > 2) {
        if (rows.count > 64) return experts_tile<ENC, 4, HILO, GATED>(p, r, rows, col_tile);
    }
    if constexpr (FM > 1) {
        if (rows.count > 32) return experts_tile<ENC, 2, HILO, GATED>(p, r, rows, col_tile);
    }
    experts_tile<ENC, 1, HILO, GATED>(p, r, rows, col_tile);
}

// ---------------------------------------------------------------------------------------------------------------------------
// the lhs
// ---------------------------------------------------------------------------------------------------------------------------
// A row by TPR threads, eight columns a thread and turn.
template <typename AT, int TPR>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void experts_prep_kernel(const AT* __restrict__ a, int64_t rows, int k, int units, int with_sums, int chunk_log, uint8_t* __restrict__ a16,
                                                                             uint8_t* __restrict__ sums, float* __restrict__ inv) {
    constexpr bool kF32 = sizeof(AT) == 4;
    constexpr int kThreads = TPR > 256 ? TPR : 256, kPer = kF32 ? 2 : 1, kHeld = 4;
    __shared__ uint32_t wmax[kThreads / 64];
    const int tid = threadIdx.x % TPR, part = threadIdx.x / TPR;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / TPR) + part;
    const bool here = row < rows;
    const AT* const ar = a + (here ? row : rows - 1) * k;
    const int pieces = k >> 3, turns = (pieces + TPR - 1) / TPR;
    LhsPiece<AT> held[kHeld];
    uint32_t top = 0;
    if (turns <= kHeld) {
#pragma unroll
        for (int i = 0; i < kHeld; i++)
            if (i < turns) held[i] = load_piece(ar + 8 * min(tid + i * TPR, pieces - 1));
#pragma unroll
        for (int i = 0; i < kHeld; i++)
            if (i < turns) top = largest_bits(top, held[i]);
    } else {
        for (int pc = tid; pc < pieces; pc += TPR) top = largest_bits(top, load_piece(ar + 8 * pc));
    }
    float mx = largest_of<AT>(top);
    if (any_not_finite(mx)) {
        mx = 0.0f;
        for (int pc = tid; pc < pieces; pc += TPR) mx = largest_finite(mx, load_piece(ar + 8 * pc));
    }
    uint32_t most = wave_max_nonneg_bits(mx);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = most;
        __syncthreads();
        most = 0;
#pragma unroll
        for (int i = 0; i < TPR / 64; i++) most = max(most, wmax[part * (TPR / 64) + i]);
    }
    if (!here) return;
    float inverse;
    const float s = row_scale(most, with_sums ? kRowTopWithSums : kRowTop, inverse);
    if (tid == 0) inv[row] = inverse;
    uint8_t* const to = a16 + row * units * (512 * kPer);
    auto emit = [&](int pc, const LhsPiece<AT>& x) __attribute__((always_inline)) {
        float v[8];
        unpack_piece(x, v);
        // columns 8 pc ..: block blk of 32, half g, step 2 blk + a: piece 2 (step within the chunk) + g
        const int blk = pc >> 2, at_g = (pc >> 1) & 1, step = 2 * blk + (pc & 1), plane = 32 << chunk_log;
        uint8_t* const at = to + (step >> chunk_log) * (plane * kPer) + (2 * (step & ((1 << chunk_log) - 1)) + at_g) * 16;
        constexpr int perm[8] = {0, 2, 1, 3, 4, 6, 5, 7};
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= s;
        HalfPack hi;
#pragma unroll
        for (int i = 0; i < 4; i++) hi.u[i] = narrow2(v[perm[2 * i]], v[perm[2 * i + 1]]);
        *(half8*)at = hi.h;
        if constexpr (kF32) {
            HalfPack lo;
            float rest[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float h = (float)hi.h[i];
                rest[i] = fabsf(h) <= 65504.0f ? v[perm[i]] - h : 0.0f;  // (an infinity has no residual: inf - inf)
            }
#pragma unroll
            for (int i = 0; i < 4; i++) lo.u[i] = narrow2(rest[2 * i], rest[2 * i + 1]);
            *(half8*)(at + plane) = lo.h;
        }
        if (with_sums) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i += 2) sum += v[i] + v[i + 1];
            sum += dpp_move<0xB1>(sum);
            sum += dpp_move<0x4E>(sum);  // the four threads of a block of 32
            if ((pc & 3) == 0) {
                const float sh = h2f(f2h(sum));
                _Float16* const sp = (_Float16*)(sums + (row * units + (blk >> 3)) * 32) + (blk & 7);
                sp[0] = (_Float16)sh;
                sp[8] = (_Float16)(sum - sh);
            }
        }
    };
    if (turns <= kHeld) {
#pragma unroll
        for (int i = 0; i < kHeld; i++)
            if (tid + i * TPR < pieces) emit(tid + i * TPR, held[i]);
    } else {
        for (int pc = tid; pc < pieces; pc += TPR) emit(pc, load_piece(ar + 8 * pc));
    }
}

// Q4_0: Q8_0 codes as fp16 (exact), block scales in the place of the sums; what a unit has beyond the row is zeros.  Four neighbouring threads hold a block.
template <typename AT>
__global__ __launch_bounds__(256) void experts_prep_q8_kernel(const AT* __restrict__ a, int64_t rows, int k, int units, uint8_t* __restrict__ a16, uint8_t* __restrict__ sums, float* __restrict__ inv) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / (units * 32);
    if (row >= rows) return;  // (whole blocks: a multiple of four threads)
    const int pc = (int)(i - row * (units * 32)), pieces = k >> 3;
    if (pc == 0) inv[row] = 1.0f;
    constexpr int kSteps = eg_steps(QMM_Q4_0);
    const int blk = pc >> 2, sub = pc & 3, g = sub & 1, step = 2 * blk + (sub >> 1);  // columns 32 blk + 16 a + 8 g: step 2 blk + a
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (pc < pieces) unpack_piece(load_piece(a + row * k + pc * 8), v);
    float mx = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(v[j]));
    mx = fmaxf(mx, dpp_move<0xB1>(mx));
    mx = fmaxf(mx, dpp_move<0x4E>(mx));
    uint16_t dh;
    const float id = q8_0_block_rule<true>(mx, dh);
    constexpr int perm[8] = {0, 2, 1, 3, 4, 6, 5, 7};
    gd_u4 o;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = pack_half2((float)q8_0_code(v[perm[2 * j]], id), (float)q8_0_code(v[perm[2 * j + 1]], id));
    *(gd_u4*)(a16 + row * units * 512 + (step / kSteps) * (32 * kSteps) + (2 * (step % kSteps) + g) * 16) = o;
    if (sub == 0) {
        uint16_t* const sp = (uint16_t*)(sums + (row * units + (blk >> 3)) * 32) + (blk & 7);
        sp[0] = dh;
        sp[8] = 0;
    }
}

struct EgSpace {
    int64_t sums, inv, bytes;  // (a16 first)
};
EgSpace eg_space(const ExpertCall& c) {
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    const int64_t units = (c.k + 255) / 256;
    EgSpace s;
    s.sums = up(c.lhs_rows * units * 512 * (c.lhs_dtype == QMM_F32 && c.encoding != QMM_Q4_0 ? 2 : 1));
    s.inv = s.sums + up(c.encoding == QMM_Q6_K ? 0 : c.lhs_rows * units * 32);
    s.bytes = s.inv + up(c.lhs_rows * 4);
    return s;
}

template <typename AT>
hipError_t run_prep(const ExpertCall& c, const EgArgs& p, hipStream_t s) {
    const AT* const a = (const AT*)c.lhs;
    uint8_t *const a16 = (uint8_t*)p.a16, *const sums = (uint8_t*)p.sums;
    float* const inv = (float*)p.inv;
    const int k = (int)c.k;
    if (c.encoding == QMM_Q4_0) {
        experts_prep_q8_kernel<AT><<<dim3((unsigned)((c.lhs_rows * p.units * 32 + 255) / 256)), dim3(256), 0, s>>>(a, c.lhs_rows, k, p.units, a16, sums, inv);
    } else {
        const int with_sums = c.encoding != QMM_Q6_K, chunk_log = eg_steps(c.encoding) == 4 ? 2 : 1;
        if (k <= 1024) experts_prep_kernel<AT, 64><<<dim3((unsigned)((c.lhs_rows + 3) / 4)), dim3(256), 0, s>>>(a, c.lhs_rows, k, p.units, with_sums, chunk_log, a16, sums, inv);
        else if (k <= 8192) experts_prep_kernel<AT, 256><<<dim3((unsigned)c.lhs_rows), dim3(256), 0, s>>>(a, c.lhs_rows, k, p.units, with_sums, chunk_log, a16, sums, inv);
        else experts_prep_kernel<AT, 1024><<<dim3((unsigned)c.lhs_rows), dim3(1024), 0, s>>>(a, c.lhs_rows, k, p.units, with_sums, chunk_log, a16, sums, inv);
    }
    return hipGetLastError();
}

int64_t eg_tiles(const Routing& r, int fm, int64_t n, bool gated) { return most_groups(r.pairs, r.experts, 32 * fm) * ((n + (gated ? 63 : 127)) / (gated ? 64 : 128)); }

template <int ENC, int FM, bool HILO, bool GATED>
hipError_t run_gemm(const EgArgs& p, const Routing& r, hipStream_t s) {
    constexpr int lds = std::max(std::max(EgLds<ENC, FM, HILO>::kBytes, EgLds<ENC, 1, HILO>::kBytes), EgLds<ENC, std::min(FM, 2), HILO>::kBytes);
    const hipError_t e = allow_full_lds<experts_gemm_kernel<ENC, FM, HILO, GATED>>();
    if (e != hipSuccess) return e;
    const int64_t tiles = eg_tiles(r, FM, p.n, GATED), part = (tiles + 7) / 8, y = std::min<int64_t>(part, 32768);
    experts_gemm_kernel<ENC, FM, HILO, GATED><<<dim3(8, (unsigned)y, (unsigned)((part + y - 1) / y)), dim3(64 * kEgWaves), lds, s>>>(p, r);
    return hipGetLastError();
}
template <int ENC, int FM, bool HILO>
hipError_t run_gemm(const EgArgs& p, const Routing& r, hipStream_t s) {
    return p.gated ? run_gemm<ENC, FM, HILO, true>(p, r, s) : run_gemm<ENC, FM, HILO, false>(p, r, s);
}
// rows of a group: 32 fm
template <int ENC, bool HILO>
hipError_t run_gemm_rows(const EgArgs& p, const Routing& r, int fm, hipStream_t s) {
    constexpr int kMost = eg_most(ENC, HILO);
    return fm == 1 ? run_gemm<ENC, 1, HILO>(p, r, s) : fm == 2 ? run_gemm<ENC, 2, HILO>(p, r, s) : run_gemm<ENC, kMost, HILO>(p, r, s);
}
template <int ENC>
hipError_t run_gemm(const EgArgs& p, const Routing& r, int fm, bool hilo, hipStream_t s) {
    if constexpr (ENC != QMM_Q4_0) {
        if (hilo) return run_gemm_rows<ENC, true>(p, r, fm, s);
    }
    return run_gemm_rows<ENC, false>(p, r, fm, s);
}

// Rows of a group, in 32s, by what an expert has on average.  Few rows: more groups fill the part better, and less is computed for rows that are not there; many: a weight is unpacked once for more of them.
// us with 32 / 64 / 128 rows, bf16 rows, 8 of 64 experts, 1024 x 2048: Q4_K 32 rows an expert 37 / 44 / 42, 64 56 / 55 / 56, 128 88 / 81 / 85, 192 120 / 104 / 105; Q6_K (two products a weight) 24 60 / 62 / 56,
// 48 85 / 65 / 74, 128 160 / 120 / 118, 192 211 / 151 / 145; 2 of 8, 14336 x 4096: Q4_K 32 106 / 103 / 103, 64 171 / 157 / 155, 256 498 / 390 / 344; fp32 rows Q4_K 48 69 / 73, 96 111 / 104.
// Q4_0 (no 128): 8 of 64, 1024 x 2048 gate and up 32 rows 50 / 55, 48 90 / 74, 64 89 / 77, 128 175 / 141; 2 of 8, 14336 x 4096 32 93 / 97, 48 154 / 130.  But a workgroup is bound by its own chain of steps: where
// tiles of 64 rows are less than one and a half a compute unit, those of 32 fill it better: 4 of 16, 1408 x 2080, drawn 64 rows (264 tiles of 64) 34 / 42, 96 (352) 42 / 43, 128 (440) 54 / 45.
int eg_rows(const ExpertCall& c, const Routing& r) {
    const int64_t mean = r.pairs / r.experts;
    const bool f32 = c.lhs_dtype == QMM_F32;
    if (c.encoding == QMM_Q4_0) return mean <= 40 || (r.pairs / 64 + r.experts / 2) * ((c.n + 127) / 128) * (c.gated ? 2 : 1) < 384 ? 1 : 2;
    const int one = !f32 && (c.encoding == QMM_Q5_K || c.encoding == QMM_Q6_K) ? 24 : 48;
    return std::min(mean <= one ? 1 : mean <= 160 ? 2 : 4, eg_most(c.encoding, f32));
}

}  // namespace

bool experts_gemm_supported(const ExpertCall& c, const Routing& r) {
    if (kernel_disabled("experts_gemm")) return false;
    const int64_t bpb = c.encoding == QMM_Q4_0 ? Q4_0_BPB : c.encoding == QMM_Q4_K ? Q4_K_BPB : c.encoding == QMM_Q5_K ? Q5_K_BPB : Q6_K_BPB, epb = c.encoding == QMM_Q4_0 ? 32 : 256;
    const int64_t blocks = c.n * (c.k / epb);
    if (blocks * bpb > 0x7fffffff || eg_tiles(r, eg_rows(c, r), c.n, c.gated) > 0x7fffffff) return false;  // (offsets in a matrix, and the tiles' numbers, have 32 bits)
    const uintptr_t all = (uintptr_t)c.w[0] | (uintptr_t)c.expert_stride[0] | (c.gated ? (uintptr_t)c.w[1] | (uintptr_t)c.expert_stride[1] : 0);
    // Q4_0: rows of whole units have to begin at multiples of four, others may begin two bytes later (an expert's, after an odd number of blocks)
    if (c.encoding == QMM_Q4_0) return (all & 1) == 0 && (((uintptr_t)c.w[0] | (c.gated ? (uintptr_t)c.w[1] : 0)) & 3) == 0 && ((all & 3) == 0 || c.k % 256 != 0);
    if (all & 3) return false;
    return c.encoding != QMM_Q6_K || blocks % 2 == 0;  // (an odd last block would be read two bytes beyond its end)
}

int64_t experts_gemm_workspace_bytes(const ExpertCall& c) { return eg_space(c).bytes; }

hipError_t launch_experts_gemm(const ExpertCall& c, const Routing& r, void* out, bool out_bf16, void* workspace, hipStream_t s) {
    const EgSpace space = eg_space(c);
    const uint8_t* const ws = (const uint8_t*)workspace;
    const EgArgs p{ws,      ws + space.sums, (const float*)(ws + space.inv), {c.w[0], c.w[1]}, {c.expert_stride[0], c.expert_stride[1]}, c.lhs_top, (int)c.n, (int)c.k, (int)((c.k + 255) / 256),
                   c.gated, out,             out_bf16};
    const hipError_t e = c.lhs_dtype == QMM_F32 ? run_prep<float>(c, p, s) : run_prep<uint16_t>(c, p, s);
    if (e != hipSuccess) return e;
    const bool hilo = c.lhs_dtype == QMM_F32;
    const int fm = eg_rows(c, r);
    switch (c.encoding) {
        case QMM_Q4_0: return run_gemm<QMM_Q4_0>(p, r, fm, hilo, s);
        case QMM_Q4_K: return run_gemm<QMM_Q4_K>(p, r, fm, hilo, s);
        case QMM_Q5_K: return run_gemm<QMM_Q5_K>(p, r, fm, hilo, s);
        default: return run_gemm<QMM_Q6_K>(p, r, fm, hilo, s);
    }
}

}  // namespace qmm
