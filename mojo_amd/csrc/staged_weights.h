// The packed weights of the GEMMs whose loads go to LDS by themselves (gemm_staged.hip, experts_gemm.hip).
#pragma once
#include "gemm_direct.h"
#include "lds_stream.h"

namespace qmm {

namespace {

// The weights of one wavefront: 32 columns, two buffers of a unit of K in LDS that only it writes (issue, a load at a time) and reads (open, before_step).
// Q4_K, Q5_K: rows as they lie in memory.
template <int ENC, bool CENTER>
struct StagedK : KQuantWeights<ENC, 1, CENTER> {
    using Base = KQuantWeights<ENC, 1, CENTER>;
    using Rows = typename Base::Rows;
    static constexpr int kLoads = Rows::kLoads;
    uint32_t stage_lds;
    const uint8_t* stage;
    __device__ __forceinline__ void init(const WeightTensors& t, int n0, int lane, uint8_t* at) {
        Base::init(t, n0, lane, at);
        stage_lds = lds_address(at);
        stage = this->mine;
    }
    template <int J>
    __device__ __forceinline__ void issue(int unit, int buf) {
        if (J * 64 + 63 < Rows::kTotal || J * 64 + this->lane_ < Rows::kTotal)
            load16_to_lds(this->rows.off[J], this->rows.w + (int64_t)unit * Rows::kRow, stage_lds + buf * Base::kStage + J * 1024);
    }
    __device__ __forceinline__ void open(int, int buf) {
        this->mine = stage + buf * Base::kStage;
        this->read_head();
    }
};

// GPTQ, plain groups, K a multiple of 256 (the packed words of a unit: 32 rows).  FLUSH as for GptqWeights.
template <int FLUSH>
struct StagedGptq : NoOffsets {
    static constexpr int kSteps = 16, kFlush = FLUSH, kPlanes = 1;
    static constexpr bool kMin = false;
    static constexpr int kBlocks = 16 / FLUSH, kHead = 20, kHeads = (kBlocks * kHead + 63) / 64;  // scale blocks a unit, 16 dwords of scales and 4 of zeros each
    static constexpr int kStage = 4096 + kHeads * 256, kLoads = 4 + kHeads;
    const uint8_t* qw;
    const uint8_t* stage;
    const uint8_t* cur;
    uint32_t stage_lds, off[4];  // off: of the lane's 16 bytes in the rows 8 j .. 8 j + 7 of a unit
    int n, lane_, zshift;
    float per_group;  // 32 / group
    const uint8_t* head[kHeads];
    uint32_t head_stride[kHeads];
    int head_block[kHeads];  // its first column of a unit, in 32s
    uint32_t words[2][2];    // of a block of 32 columns
    uint32_t top0 = code_top(0x64006400u), top1 = code_top(0x54005400u);
    uint32_t s_raw[kBlocks], z_raw[kBlocks];

    __device__ __forceinline__ void init(const WeightTensors& t, int n0, int lane, uint8_t* at) {
        qw = t.w;
        stage = at;
        stage_lds = lds_address(at);
        n = t.n;
        lane_ = lane;
        zshift = 4 * (lane & 7);
        per_group = 32.0f / (float)t.group;
        // LDS row p holds word row 4 blk + 2 g + a with p = 4 blk + 2 a + g: the two half wavefronts read other banks
        const int p = lane >> 3, row = (p & 4) + 2 * (p & 1) + ((p >> 1) & 1);
#pragma unroll
        for (int j = 0; j < 4; j++) off[j] = (uint32_t)(row + 8 * j) * (uint32_t)n * 4u + (uint32_t)min(n0 + 4 * (lane & 7), n - 4) * 4u;
#pragma unroll
        for (int j = 0; j < kHeads; j++) {
            const int i = j * 64 + lane, blk = min(i / kHead, kBlocks - 1), part = i % kHead;
            head_block[j] = blk * (FLUSH / 2);
            head[j] = part < 16 ? (const uint8_t*)t.scales + min(n0 + 2 * part, n - 2) * 2 : (const uint8_t*)t.qzeros + min((n0 >> 3) + part - 16, (n >> 3) - 1) * 4;
            head_stride[j] = part < 16 ? (uint32_t)n * 2u : (uint32_t)(n >> 3) * 4u;
        }
    }
    template <int J>
    __device__ __forceinline__ void issue(int unit, int buf) {
        const uint32_t to = stage_lds + buf * kStage;
        if constexpr (J < 4) {
            load16_to_lds(off[J], qw + (int64_t)(32 * unit) * n * 4, to + J * 1024);
        } else {
            // (a group is a whole number of 32s and K below 2^27: half of one keeps the product off the integers by more than its rounding)
            const int group = (int)(((float)(8 * unit + head_block[J - 4]) + 0.5f) * per_group);
            load4_to_lds(head[J - 4] + (uint64_t)(uint32_t)group * head_stride[J - 4], to + 4096 + (J - 4) * 256);
        }
    }
    __device__ __forceinline__ void read_words(int blk) {
#pragma unroll
        for (int a = 0; a < 2; a++) words[blk & 1][a] = *(const uint32_t*)(cur + (4 * blk + 2 * a) * 128 + lane_ * 4);
    }
    __device__ __forceinline__ void open(int, int buf) {
        cur = stage + buf * kStage;
        read_words(0);
#pragma unroll
        for (int i = 0; i < kBlocks; i++) {
            s_raw[i] = *(const uint16_t*)(cur + 4096 + i * 80 + 2 * (lane_ & 31));
            z_raw[i] = *(const uint32_t*)(cur + 4096 + i * 80 + 64 + 4 * ((lane_ & 31) >> 3));
        }
    }
    template <int T>
    __device__ __forceinline__ void before_step() {
        if constexpr ((T & 1) == 0 && T < 14) read_words((T >> 1) + 1);
    }
    template <int T>
    __device__ __forceinline__ void step(int, half8 (&b)[1]) const {
        const uint32_t z = ((z_raw[T / FLUSH] >> zshift) & 0xFu) + 1u;
        const uint32_t m0 = 0xE400E400u | (z * 0x00010001u), m1 = 0xD400D400u | (z * 0x00100010u);
        const uint32_t x = words[(T >> 1) & 1][T & 1], y = x >> 8;
        b[0] = pack4(pk_add((x & 0x000F000Fu) | top0, m0), pk_add((x & 0x00F000F0u) | top1, m1), pk_add((y & 0x000F000Fu) | top0, m0), pk_add((y & 0x00F000F0u) | top1, m1));
    }
    template <int I>
    __device__ __forceinline__ float scale_at() const { return h2f((uint16_t)s_raw[I]); }
};

// Q6_K in a tensor that begins at a multiple of four: blocks of 210 bytes lie at even addresses, loads to LDS want multiples of four: a row's 212 bytes from the last such address on, 208 of them in pieces
// of 16, the last four apart.  The fields begin `skew` (0 or 2) bytes later, other in every row and unit.  With an even number of blocks the last one of the matrix
// begins at 2 mod 4 and ends with those four bytes; an odd number of them, whose last would be read two bytes beyond its end, is not this kernel's (staged_plan).
template <int FLUSH>
struct StagedQ6 : Q6Weights<1, FLUSH> {
    using Base = Q6Weights<1, FLUSH>;
    static constexpr int kPieces = 13, kTotal = 32 * kPieces, kWide = (kTotal + 63) / 64, kLoads = kWide + 1, kTail = kTotal * 16, kStage = kTail + 128;
    const uint8_t* w;
    const uint8_t* stage;
    const uint8_t* cur;
    uint32_t stage_lds, off[kWide], off_tail;
    const uint8_t* tail;
    uint32_t odd, skew, mine_odd;  // odd: bit 1 + j: the row of piece j begins at 2 mod 4 in even units; mine_odd: the lane's own row, bit 1
    __device__ __forceinline__ void init(const WeightTensors& t, int n0, int lane, uint8_t* at) {
        this->g = lane >> 5;
        this->lane_ = lane;
        w = t.w;
        stage = at;
        stage_lds = lds_address(at);
        const uint32_t row_bytes = (uint32_t)(t.k / 256 * Q6_K_BPB);
        auto row_at = [&](int row) __attribute__((always_inline)) { return (uint32_t)min(n0 + row, t.n - 1) * row_bytes; };
        odd = 0;
#pragma unroll
        for (int j = 0; j < kWide; j++) {
            const int i = min(j * 64 + lane, kTotal - 1), row = i / kPieces;
            off[j] = row_at(row) + 16 * (i - row * kPieces);
            odd |= (row_at(row) & 2u) << j;
        }
        off_tail = row_at(lane & 31) + 208;
        mine_odd = row_at(lane & 31) & 2u;
    }
    template <int J>
    __device__ __forceinline__ void issue(int unit, int buf) {
        const uint8_t* b = w + (int64_t)unit * Q6_K_BPB;
        const uint32_t o = (unit & 1) ? ~odd : odd, to = stage_lds + buf * kStage;
        if constexpr (J < kWide) {
            if (J * 64 + 63 < kTotal || J * 64 + this->lane_ < kTotal) load16_to_lds(off[J] + 2 - ((o >> J) & 2u), b - 2, to + J * 1024);
        } else if (this->lane_ < 32) {
            load4_to_lds(b - 2 + (off_tail + 2 - ((mine_odd ^ (unit << 1)) & 2u)), to + kTail);
        }
    }
    // 16 bytes at offset `at` of the block
    __device__ __forceinline__ gd_u4 field(int at) const {
        const gd_u4 v = *(const gd_u4*)(cur + at);
        const uint32_t e = *(const uint32_t*)(at == 192 ? tail : cur + at + 16);
        return gd_u4{__builtin_amdgcn_alignbyte(v.y, v.x, skew), __builtin_amdgcn_alignbyte(v.z, v.y, skew), __builtin_amdgcn_alignbyte(v.w, v.z, skew),
                     __builtin_amdgcn_alignbyte(e, v.w, skew)};
    }
    __device__ __forceinline__ void read_half(int h) {
        this->ql[0][0] = field(64 * h + 16 * this->g);
        this->ql[0][1] = field(64 * h + 32 + 16 * this->g);
        this->qh[0] = field(128 + 32 * h + 16 * this->g);
    }
    __device__ __forceinline__ void open(int unit, int buf) {
        const uint8_t* b = stage + buf * kStage;
        cur = b + (this->lane_ & 31) * 208;
        tail = b + kTail + 4 * (this->lane_ & 31);
        skew = (mine_odd ^ (unit << 1)) & 2u;
        read_half(0);
        const gd_u4 s = field(192);
        const uint32_t sel = this->g ? 0x07050301u : 0x06040200u;
        this->sc[0][0] = __builtin_amdgcn_perm(s.y, s.x, sel);
        this->sc[0][1] = __builtin_amdgcn_perm(s.w, s.z, sel);
        this->d[0] = (*(const uint32_t*)tail >> (8 * skew)) & 0xffffu;
    }
    template <int T>
    __device__ __forceinline__ void before_step() {
        if constexpr (T == 7) read_half(1);
    }
};

template <int ENC, int FLUSH, bool CENTER>
using StagedOf = std::conditional_t<ENC == QMM_GPTQ, StagedGptq<FLUSH>, std::conditional_t<ENC == QMM_Q6_K, StagedQ6<FLUSH>, StagedK<ENC == QMM_Q5_K ? QMM_Q5_K : QMM_Q4_K, CENTER>>>;

}  // namespace

}  // namespace qmm
