// Log probabilities of given tokens, entropy and the largest alternatives of rows of logits, in one pass over them.
//
//   m = max x, S = sum exp(x - m), t = sum (x - m) exp(x - m):   log p(i) = x_i - m - log S,   H = log S - t / S
//
// The elements equal to the running maximum are counted (c) and kept out of the sum (s), so that S = c + s and log S = log1p(c - 1 + s): a row whose
// largest value holds all but 1e-6 of the mass has a log probability of 1e-6, not of what fp32 leaves of 1 + 1e-6.  c is a number, so counting it takes no rounding either.
// An element costs one multiply-add, one exponential (four times an ordinary instruction), a sum, a multiply-add for t and a clamp that makes 0 x -inf a 0: exp(x - m) is 2^(x L - f) with L = log2 e and
// f = m L rounded; what that rounding moved, the same for every element, is put right where the wavefronts are joined.
// Parts of a row (lanes, wavefronts, workgroups) each have their (m, c, s, t) and are joined with exp(m_i - m).
//
// Alternatives.  A value that is among the `top` largest lies in one of the `top` runs of neighbouring values (four lanes' loads: 16 fp32 or 32 bf16 values) with the largest maxima, equal ones by
// rising index.  So the pass leaves the maximum of every run in LDS (two DPP steps a load), and what follows looks for the largest of few: of 16 runs together,
// of the runs of the chosen ones, of the values of the chosen runs.  A key is the value's bits in an order that integers compare right, above the index inverted: equal values by rising index, no two keys alike.
// The time of this long way does not depend on the values, where a list that every larger value is put into takes a row in rising order apart.  Up to 32 alternatives there is a shorter one for nearly all rows
// (sort_gathered): one row of 128256 14.4 -> 12.5 us, 1021 bf16 rows 68 -> 65.
//
// What bounds it: with many rows the loads (a row is read once; the chosen runs again, from L2).  With few, the way through two launches: parts of a row go to several workgroups until
// they are enough for the part, and one workgroup a row joins them (lp_plan).  1021 rows of 128256 bf16, 5 alternatives:
// 64 us, 4.1 TB/s, vector units busy 0.86 of the time; 200 rows fp32 22 us, 4.6 TB/s; one row, 20 alternatives: 12.6 us.
#include <algorithm>

#include "experts.h"

namespace qmm {

namespace {

constexpr int kLpThreads = 512, kLpWaves = kLpThreads / 64;
constexpr int kLpLoads = 4;           // 16-byte loads of a lane at once
constexpr int kLpStep = kLpThreads * kLpLoads;  // loads of a workgroup at once
constexpr int kLpRuns = 8192;         // runs of a workgroup at most (LDS: 32 KB)

struct LpState {
    float m, s, t;
    int c;
};

typedef uint32_t lp_u4 __attribute__((ext_vector_type(4)));

// Larger values have larger numbers; -0 is 0, NaN is below everything.  Never 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 1u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) { return (uint64_t)order_of(x) << 32 | (uint32_t)~index; }
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return ~(uint32_t)key; }
__device__ __forceinline__ float value_of(uint64_t key) {  // (a NaN comes out as one)
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}

constexpr float kLog2e = 1.44269504088896f, kLn2 = 0.693147180559945f;
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }  // d <= 0
// what stands for -inf where it meets a factor of exp(-inf) = 0
constexpr float kLpFloor = -150.0f;
// Beyond, the next fp32 number is 128 lower and its exponential 0, as that of all others (f = inf); up to here the rounding of m L is no more than 64, and 2 to that power a number.
constexpr float kLpFar = 1073741824.0f;

// b joins a.  (m = -inf: nothing but -inf so far, whose number does not matter.)
__device__ __forceinline__ void join(LpState& a, const LpState& b) {
    const bool more = b.m > a.m, even = b.m == a.m;
    const float lm = more ? a.m : b.m, ls = more ? a.s : b.s, lt = more ? a.t : b.t, hs = more ? b.s : a.s, ht = more ? b.t : a.t;
    const int lc = more ? a.c : b.c, hc = more ? b.c : a.c;
    a.m = more ? b.m : a.m;
    const float d = fmaxf(lm - a.m, kLpFloor), f = exp_of(d), n = (float)lc + ls;
    a.c = even ? hc + lc : hc;
    a.s = even ? hs + ls : fmaf(f, n, hs);
    a.t = even ? ht + lt : fmaf(f, fmaf(d, n, lt), ht);
}

// The value of lane ^ MASK, without LDS: DPP within 16 lanes (4: mirrored in eight, then in four), exchanges of rows beyond.
template <int MASK>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int lane) {
    if constexpr (MASK == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);
    if constexpr (MASK == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);
    if constexpr (MASK == 4) return (uint32_t)__builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true), 0x1B, 0xf, 0xf, true);
    if constexpr (MASK == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true);
    if constexpr (MASK == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (lane & 16) ? r[0] : r[1];
    }
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (lane & 32) ? r[0] : r[1];
}
template <int MASK>
__device__ __forceinline__ float lane_xor(float v, int lane) { return __uint_as_float(lane_xor<MASK>(__float_as_uint(v), lane)); }
template <int MASK = 32>
__device__ __forceinline__ void wave_join(LpState& a, int lane) {
    const LpState b{lane_xor<MASK>(a.m, lane), lane_xor<MASK>(a.s, lane), lane_xor<MASK>(a.t, lane), (int)lane_xor<MASK>((uint32_t)a.c, lane)};
    join(a, b);
    if constexpr (MASK > 1) wave_join<MASK / 2>(a, lane);
}

// One step of a bitonic sort over the lanes: the larger of a pair to the lane that wants it.
template <int MASK>
__device__ __forceinline__ void exchange(float& v, int lane, bool larger) {
    const float o = lane_xor<MASK>(v, lane);
    v = larger ? fmaxf(v, o) : fminf(v, o);
}
template <int MASK>
__device__ __forceinline__ void exchange(uint64_t& v, int lane, bool larger) {
    const uint64_t o = (uint64_t)lane_xor<MASK>((uint32_t)(v >> 32), lane) << 32 | lane_xor<MASK>((uint32_t)v, lane);
    v = (v > o) == larger ? v : o;
}
template <int SIZE, int MASK, typename V>
__device__ __forceinline__ void merge_step(V& v, int lane) {
    exchange<MASK>(v, lane, ((lane & MASK) == 0) == (SIZE == 64 || (lane & SIZE) == 0));
    if constexpr (MASK > 1) merge_step<SIZE, MASK / 2>(v, lane);
}
template <int SIZE = 2, int COUNT = 64, typename V>
__device__ __forceinline__ void sort64(V& v, int lane) {  // falling; the first COUNT lanes
    merge_step<SIZE, SIZE / 2>(v, lane);
    if constexpr (SIZE < COUNT) sort64<SIZE * 2, COUNT>(v, lane);
}
// a: falling; reversed: another falling list, last entry first.  The 64 largest of both, falling.
__device__ __forceinline__ void merge64(uint64_t& a, uint64_t reversed, int lane) {
    a = a > reversed ? a : reversed;
    merge_step<64, 32>(a, lane);
}

// The lists of the workgroup's wavefronts (falling, one entry a lane) to one, in lists[0 .. 63] (visible to all afterwards).
template <int WAVES>
__device__ __forceinline__ void merge_waves(uint64_t& mine, uint64_t* lists, int wave, int lane) {
    __syncthreads();  // (whoever still reads the lists of before)
    lists[wave * 64 + lane] = mine;
#pragma unroll
    for (int half = WAVES / 2; half; half >>= 1) {
        __syncthreads();
        if (wave < half) {
            merge64(mine, lists[(wave + half) * 64 + 63 - lane], lane);
            lists[wave * 64 + lane] = mine;
        }
    }
    __syncthreads();
}
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) { return (uint64_t)(uint32_t)__shfl((int)(v >> 32), lane) << 32 | (uint32_t)__shfl((int)v, lane); }
// The `top` largest of key(0) .. key(count - 1) (0: none) first in lists[0 .. 63].  (key is called by whole wavefronts.)
template <int WAVES, typename F>
__device__ __forceinline__ void top_keys(int count, int top, uint64_t* lists, int wave, int lane, F&& key) {
    uint64_t mine = 0;
    for (int at = wave * 64; at < count; at += WAVES * 64) {
        uint64_t v = key(min(at + lane, count - 1));
        if (at + lane >= count) v = 0;
        if (at == wave * 64) {
            sort64(v, lane);
            mine = v;
        } else if (__any(v > shfl64(mine, top - 1))) {
            sort64(v, lane);
            merge64(mine, shfl64(v, 63 - lane), lane);
        }
    }
    merge_waves<WAVES>(mine, lists, wave, lane);
}

// Nearly always there is a shorter way: of 64 numbers, each the largest of a share of the values, the top-th largest is a bound that at least `top` values reach, and hardly more (20 of them: 24 at random).
// Those that do are gathered in any order and sorted once.  With more than kLpFew wanted the bound lets too many through; if more than 64 reach it (values that are equal, a mask), the long way is taken.
constexpr int kLpFew = 32;
// The gathered keys, falling, in lists[0 .. 63]; false: there were too many.
__device__ __forceinline__ bool sort_gathered(uint64_t* lists, const int* taken, int wave, int lane) {
    __syncthreads();
    const int count = *taken;
    if (count > 64) return false;
    if (wave == 0) {
        uint64_t v = lane < count ? lists[lane] : 0;
        if (count <= 8) sort64<2, 8>(v, lane);
        else if (count <= 32) sort64<2, 32>(v, lane);
        else sort64(v, lane);
        lists[lane] = v;
    }
    __syncthreads();
    return true;
}

// The largest of three (no NaN among the results unless all are); the compiler's own would first make each value a quiet one.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// A row as 16-byte loads at multiples of 16 bytes: load v holds the values v * kPer - skew .. of the row; the first and the last one may hold fewer.
template <typename T>
struct LpRow {
    static constexpr int kPer = 16 / sizeof(T);
    const T* aligned;
    int skew, vocab;
    __device__ __forceinline__ LpRow(const T* row, int v) : vocab(v) {
        skew = (int)(((uintptr_t)row & 15) / sizeof(T));
        aligned = row - skew;
    }
    __device__ __forceinline__ int loads() const { return (skew + vocab + kPer - 1) / kPer; }
    __device__ __forceinline__ bool whole(int v) const { return v * kPer >= skew && (v + 1) * kPer - skew <= vocab; }
    static __device__ __forceinline__ void unpack(const lp_u4& raw, float (&x)[kPer]) {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(raw[i]);
            else x[i] = __uint_as_float((i & 1) ? raw[i >> 1] & 0xffff0000u : raw[i >> 1] << 16);
        }
    }
    // load v; -inf in the place of values that the row does not have
    __device__ __forceinline__ lp_u4 edge(int v) const {
        lp_u4 raw;
        T e[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int at = v * kPer + i - skew;
            if constexpr (sizeof(T) == 4) e[i] = at >= 0 && at < vocab ? aligned[(int64_t)v * kPer + i] : -__builtin_inff();
            else e[i] = at >= 0 && at < vocab ? aligned[(int64_t)v * kPer + i] : (T)0xff80;
        }
        __builtin_memcpy(&raw, e, 16);
        return raw;
    }
    __device__ __forceinline__ float at(int64_t i) const { return load_f32(aligned, i + skew); }
};

struct LpOut {
    const void* tokens;  // null: none
    int wide, per_row;   // 64-bit tokens; tokens of a row
    float *chosen, *entropy, *top_values;
    int32_t* top_ids;
    int top;
};

// A token of a row and its logit, asked for before the row is looked at.
struct LpToken {
    int64_t token;
    float x;
};
template <typename T>
__device__ __forceinline__ LpToken token_at(int64_t row_number, const LpRow<T>& row, int i, const LpOut& out) {
    const int64_t at = row_number * out.per_row + i, token = out.wide ? ((const int64_t*)out.tokens)[at] : ((const int32_t*)out.tokens)[at];
    return {token, token >= 0 && token < row.vocab ? row.at(token) : 0.0f};
}
// What a row's state says.  mine: the thread's token (the first `blockDim` of the row's have one each); lists: the row's `top` largest keys.
template <typename T>
__device__ __forceinline__ void finish_row(int64_t row_number, const LpRow<T>& row, const LpState& a, LpToken mine, const uint64_t* lists, const LpOut& out) {
    const float rest = (float)(a.c - 1) + a.s, log_total = log1pf(rest);
    const bool none = a.m == -__builtin_inff() && !(a.s != a.s);  // no mass at all
    const float bad = a.m == __builtin_inff() ? __builtin_nanf("") : 0.0f;
    auto log_p = [&](float x) { return none ? -__builtin_inff() : (x - a.m) - log_total + bad; };
    for (int i = threadIdx.x; i < out.per_row; i += (int)blockDim.x) {
        if (i >= (int)blockDim.x) mine = token_at(row_number, row, i, out);
        out.chosen[row_number * out.per_row + i] = mine.token < 0 ? 0.0f : mine.token >= row.vocab ? __builtin_nanf("") : log_p(mine.x);
    }
    if (threadIdx.x == 0) out.entropy[row_number] = none ? 0.0f : log_total - a.t / ((float)a.c + a.s) + bad;
    if ((int)threadIdx.x < out.top) {
        const uint64_t key = lists[threadIdx.x];
        out.top_ids[row_number * out.top + threadIdx.x] = (int32_t)index_of(key);
        out.top_values[row_number * out.top + threadIdx.x] = log_p(value_of(key));
    }
}

// A part of a row: `per` loads (a multiple of four) of it; parts: workgroups of a row.  One: the row is finished here.
template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprobs_kernel(const T* __restrict__ logits, int64_t stride, int vocab, int per, int parts, LpState* __restrict__ states,
                                                              uint64_t* __restrict__ keys, LpOut out) {
    constexpr int kPer = LpRow<T>::kPer, kRun = 4 * kPer;  // values of a load, of a run
    extern __shared__ __attribute__((aligned(16))) float runs[];
    __shared__ uint64_t lists[kLpThreads];
    __shared__ LpState waves[kLpWaves];
    __shared__ int picked, taken;
    if (threadIdx.x == 0) picked = taken = 0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), part = (int)blockIdx.y;
    const int64_t row_number = blockIdx.x;
    const LpRow<T> row(logits + row_number * stride, vocab);
    const int first = part * per, end = min(first + per, row.loads());
    const bool wanted = out.top > 0;
    LpToken token{0, 0.0f};
    if (parts == 1 && (int)threadIdx.x < out.per_row) token = token_at(row_number, row, threadIdx.x, out);

    const int whole0 = row.skew ? 1 : 0, whole1 = min(end, (row.skew + vocab) / kPer);  // loads that the row fills
    float m = -__builtin_inff(), f = 0.0f, s = 0.0f, t = 0.0f;  // m and f = m L: of the wavefront; s and t (in units of log 2): of the lane
    int c = 0;                                                  // of the wavefront
    auto take = [&](int v0, const lp_u4 (&raw)[kLpLoads]) __attribute__((always_inline)) {
        float x[kLpLoads][kPer], most[kLpLoads], all = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < kLpLoads; j++) {
            LpRow<T>::unpack(raw[j], x[j]);
            most[j] = x[j][kPer - 1];
#pragma unroll
            for (int i = 0; i + 1 < kPer - 1; i += 2) most[j] = max3(most[j], x[j][i], x[j][i + 1]);
            most[j] = fmaxf(most[j], x[j][kPer - 2]);
            all = fmaxf(all, most[j]);
        }
        if (wanted) {
            // the maximum of a run, four lanes, is in all of them; lane j of four keeps that of load j
            float keep = 0.0f;
#pragma unroll
            for (int j = 0; j < kLpLoads; j++) {
                float q = fmaxf(most[j], dpp_move<0xB1>(most[j]));
                q = fmaxf(q, dpp_move<0x4E>(q));
                keep = (lane & 3) == j ? q : keep;
            }
            const int run = ((v0 - first) >> 2) + (lane & 3) * 16 + (lane >> 2);
            if (run * 4 < end - first) runs[run] = keep;
        }
        if (__any(all >= m)) {
            // a new maximum, or one equal to it
            float now = fmaxf(all, m);
            now = fmaxf(now, lane_xor<32>(now, lane));
            now = fmaxf(now, lane_xor<16>(now, lane));
            now = fmaxf(now, lane_xor<8>(now, lane));
            now = fmaxf(now, lane_xor<4>(now, lane));
            now = fmaxf(now, lane_xor<2>(now, lane));
            now = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(fmaxf(now, lane_xor<1>(now, lane)))));
            if (now > m) {
                // (what was the maximum is none now: c elements of 2^(m L - f))
                const float g = fabsf(now) > kLpFar ? __builtin_inff() : now * kLog2e;
                if (m > -__builtin_inff() && f < __builtin_inff()) {
                    const float d = fmaxf(f - g, 1.5f * kLpFloor), by = __builtin_amdgcn_exp2f(d), r = fmaf(m, kLog2e, -f), n = lane == 0 ? (float)c * __builtin_amdgcn_exp2f(r) : 0.0f;
                    t = by * (fmaf(d, s, t) + (d + r) * n);
                    s = by * (s + n);
                }
                m = now;
                f = g;
                c = 0;
            }
#pragma unroll
            for (int j = 0; j < kLpLoads; j++)
#pragma unroll
                for (int i = 0; i < kPer; i++) {
                    const bool is = x[j][i] == m;
                    c += (int)__popcll(__ballot(is));
                    x[j][i] = is ? -__builtin_inff() : x[j][i];
                }
        }
        float s2[2] = {0.0f, 0.0f}, t2[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kLpLoads; j++)
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                const float d = fmaf(x[j][i], kLog2e, -f), e = __builtin_amdgcn_exp2f(d);
                s2[i & 1] += e;
                t2[i & 1] = fmaf(fmaxf(d, 1.5f * kLpFloor), e, t2[i & 1]);
            }
        s += s2[0] + s2[1];
        t += t2[0] + t2[1];
    };
    // this wavefront's steps: those that the row fills, each asked for while the one before is looked at; then the first and the last, which it may not fill
    const int v_first = first + wave * 64 * kLpLoads;
    auto fills = [&](int v0) __attribute__((always_inline)) { return v0 >= whole0 && v0 + 64 * kLpLoads <= whole1; };
    int v0 = v_first < whole0 ? v_first + kLpStep : v_first;
    if (fills(v0)) {
        lp_u4 next[kLpLoads];
        auto load = [&](int v) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < kLpLoads; j++) next[j] = *(const lp_u4*)(row.aligned + (int64_t)(v + j * 64 + lane) * kPer);
        };
        load(v0);
        while (fills(v0)) {
            lp_u4 raw[kLpLoads];
#pragma unroll
            for (int j = 0; j < kLpLoads; j++) raw[j] = next[j];
            load(fills(v0 + kLpStep) ? v0 + kLpStep : v0);
            take(v0, raw);
            v0 += kLpStep;
        }
    }
#pragma unroll 1
    for (int edge = 0; edge < 2; edge++) {
        const int v_edge = edge ? v0 : v_first;
        if (v_edge >= end || (edge == 0 && v_first >= whole0)) continue;
        constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
        const lp_u4 none{kNone, kNone, kNone, kNone};
        lp_u4 raw[kLpLoads];
        const bool some = whole0 < (row.skew + vocab) / kPer;  // there is a load that the row fills, which lanes without one ask for
#pragma unroll
        for (int j = 0; j < kLpLoads; j++) {
            const int v = v_edge + j * 64 + lane;
            raw[j] = some ? *(const lp_u4*)(row.aligned + (int64_t)(v < end && row.whole(v) ? v : whole0) * kPer) : none;
        }
#pragma unroll
        for (int j = 0; j < kLpLoads; j++) {
            const int v = v_edge + j * 64 + lane;
            if (v >= end || !row.whole(v)) raw[j] = none;
        }
#pragma unroll 1
        for (int j = 0; j < kLpLoads; j++) {
            const int v = v_edge + j * 64 + lane;
            if (v >= end || row.whole(v)) continue;
            const lp_u4 one = row.edge(v);
#pragma unroll
            for (int i = 0; i < kLpLoads; i++) raw[i] = i == j ? one : raw[i];
        }
        take(v_edge, raw);
    }
    // f is m L but for its rounding r: every element was 2^r times what it is, with r more in its exponent
    const float r = fabsf(m) <= kLpFar ? fmaf(m, kLog2e, -f) : 0.0f, by = __builtin_amdgcn_exp2f(-r);
    LpState a{m, s * by, (t - r * s) * by * kLn2, lane == 0 ? c : 0};
    wave_join(a, lane);
    if (lane == 0) waves[wave] = a;
    __syncthreads();
    a = waves[0];
#pragma unroll
    for (int w = 1; w < kLpWaves; w++) {
        const LpState b = waves[w];
        join(a, b);
    }
    const int count = (end - first + 3) / 4;  // runs of this part
    bool found = !wanted;
    if (wanted && out.top <= kLpFew && count >= 64 && a.s == a.s) {
        // run r belongs to share r mod 64
        float* const shares = (float*)(lists + kLpThreads / 2);
        float most = -__builtin_inff();
        for (int run = threadIdx.x; run < count; run += kLpThreads) most = fmaxf(most, runs[run]);
        shares[threadIdx.x] = most;
        __syncthreads();
        most = shares[lane];
#pragma unroll
        for (int w = 1; w < kLpWaves; w++) most = fmaxf(most, shares[w * 64 + lane]);
        sort64(most, lane);
        const float bound = __shfl(most, out.top - 1);
        // the runs that reach it, then their values, a load a thread
        if (bound > -__builtin_inff()) {
            for (int run = threadIdx.x; run < count && *(volatile int*)&picked <= 64; run += kLpThreads) {
                if (runs[run] < bound) continue;
                const int at = atomicAdd(&picked, 1);
                if (at < 64) ((int*)(lists + 64))[at] = run;
            }
        } else if (threadIdx.x == 0) {
            picked = 65;  // (every value does)
        }
        __syncthreads();
        const int v = picked <= 64 && (int)threadIdx.x < 4 * picked ? first + 4 * ((int*)(lists + 64))[threadIdx.x >> 2] + (int)(threadIdx.x & 3) : end;
        if (v < end) {
            float x[kPer];
            LpRow<T>::unpack(row.whole(v) ? *(const lp_u4*)(row.aligned + (int64_t)v * kPer) : row.edge(v), x);  // (-inf where the row has no value)
            int reached = 0;
#pragma unroll
            for (int i = 0; i < kPer; i++) reached += x[i] >= bound;
            int at = reached ? atomicAdd(&taken, reached) : 0;
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                if (!(x[i] >= bound)) continue;
                if (at < 64) lists[at] = key_of(x[i], (uint32_t)(v * kPer + i - row.skew));
                at++;
            }
        }
        found = picked <= 64 && sort_gathered(lists, &taken, wave, lane);
    }
    if (!found) {
        if (a.s != a.s) {
            // There is a NaN.  (One that signals would have hidden its neighbours from the maxima above.)
            for (int run = threadIdx.x; run < count; run += kLpThreads) {
                float most = __builtin_nanf("");
                for (int i = 0; i < kRun; i++) {
                    const int64_t at = (first + (int64_t)run * 4) * kPer + i - row.skew;
                    if (at >= 0 && at < vocab && order_of(row.at(at)) > order_of(most)) most = row.at(at);
                }
                runs[run] = most;
            }
            __syncthreads();
        }
        int chosen;
        if (count > kLpThreads) {
            // sixteen runs together, then the runs of the chosen sixteens
            top_keys<kLpWaves>((count + 15) / 16, out.top, lists, wave, lane, [&](int i) {
                float w = runs[16 * i];
#pragma unroll
                for (int j = 1; j < 16; j++) w = fmaxf(w, runs[min(16 * i + j, count - 1)]);
                return key_of(w, (uint32_t)i);
            });
            const uint64_t sixteens = lists[lane];
            chosen = min(out.top, (count + 15) / 16);
            top_keys<kLpWaves>(chosen * 16, out.top, lists, wave, lane, [&](int i) {
                const int run = (int)index_of(shfl64(sixteens, i >> 4)) * 16 + (i & 15);
                return run < count ? key_of(runs[run], (uint32_t)run) : 0;
            });
        } else {
            top_keys<kLpWaves>(count, out.top, lists, wave, lane, [&](int i) { return key_of(runs[i], (uint32_t)i); });
        }
        const uint64_t best = lists[lane];
        chosen = min(out.top, count);
        top_keys<kLpWaves>(chosen * kRun, out.top, lists, wave, lane, [&](int i) {
            const int64_t at = (first + (int64_t)index_of(shfl64(best, i / kRun)) * 4) * kPer + i % kRun - row.skew;  // of the row
            return at >= 0 && at < vocab && at < (int64_t)end * kPer - row.skew ? key_of(row.at(at), (uint32_t)at) : 0;
        });
    }
    if (parts == 1) return finish_row(row_number, row, a, token, lists, out);
    const int64_t place = row_number * parts + part;
    if (threadIdx.x == 0) states[place] = a;
    if ((int)threadIdx.x < out.top) keys[place * out.top + threadIdx.x] = lists[threadIdx.x];
}

// The parts of a row, in their order.
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void logprobs_join_kernel(const T* __restrict__ logits, int64_t stride, int vocab, int parts, const LpState* __restrict__ states,
                                                                          const uint64_t* __restrict__ keys, LpOut out) {
    __shared__ uint64_t lists[64 * WAVES];
    __shared__ int taken;
    if (WAVES > 1) {
        if (threadIdx.x == 0) taken = 0;
        __syncthreads();
    }
    const int lane = threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int64_t row_number = blockIdx.x;
    const LpRow<T> row(logits + row_number * stride, vocab);
    LpToken token{0, 0.0f};
    if ((int)threadIdx.x < out.per_row) token = token_at(row_number, row, threadIdx.x, out);
    LpState a{-__builtin_inff(), 0.0f, 0.0f, 0};
    for (int i = lane; i < parts; i += 64) {
        const LpState b = states[row_number * parts + i];
        join(a, b);
    }
    wave_join(a, lane);
    if (out.top > 0) {
        constexpr int kLists = 64 / WAVES > 8 ? 8 : 64 / WAVES;  // parts <= kLists WAVES
        const uint64_t* const mine_of_row = keys + row_number * parts * out.top;
        bool found = false;
        if constexpr (WAVES > 1) {
            if (out.top <= kLpFew && parts >= out.top) {
                // the parts' largest
                const int all = parts * out.top;
                uint64_t v[kLpFew * 64 / (64 * WAVES)], most = lane < parts ? mine_of_row[lane * out.top] : 0;
#pragma unroll
                for (int i = 0; i < (int)(sizeof(v) / 8); i++) {
                    const int at = (int)threadIdx.x + i * 64 * WAVES;
                    v[i] = at < all ? mine_of_row[at] : 0;
                }
                sort64(most, lane);
                const uint64_t bound = shfl64(most, out.top - 1);
                if (bound) {
#pragma unroll
                    for (int i = 0; i < (int)(sizeof(v) / 8); i++)
                        if (v[i] >= bound) {
                            const int at = atomicAdd(&taken, 1);
                            if (at < 64) lists[at] = v[i];
                        }
                } else if (threadIdx.x == 0) {
                    taken = 65;
                }
                found = sort_gathered(lists, &taken, wave, lane);
            }
        }
        if (!found) {
            uint64_t v[kLists];
#pragma unroll
            for (int i = 0; i < kLists; i++) {
                const int part = wave + i * WAVES, at = i == 0 ? lane : 63 - lane;
                v[i] = part < parts && at < out.top ? mine_of_row[part * out.top + at] : 0;
            }
            uint64_t mine = v[0];
#pragma unroll
            for (int i = 1; i < kLists; i++)
                if (wave + i * WAVES < parts) merge64(mine, v[i], lane);
            merge_waves<WAVES>(mine, lists, wave, lane);
        }
    }
    finish_row(row_number, row, a, token, lists, out);
}

struct LpPlan {
    int per, parts;
};
constexpr int64_t kLpRows = 1 << 22;  // rows of a launch (a grid has up to 2^32 threads); more take one after the other, with the same plan
// Workgroups a row: as few as make the runs of one fit its LDS (33 for QMM_MAX_VOCAB fp32 values).  Beyond, one where a row is less than four steps of a workgroup (a second launch is 4 us, a step one), and
// else until there is one for each compute unit, each with a load for every thread; 64 at most.  us with 1 / 2 / 8 / 32 workgroups a row, fp32, 5 alternatives: 1 row of 32000 11.1 / 12.4 / 12.0 / 13.2, of 65536
// 15.2 / 14.7 / 12.7 / 12.3, of 128256 21.8 / 18.8 / 14.3 / 12.3; 32 rows of 128256 23.5 / 20.8 / 16.4 / 21.2; 400 rows 48.1 / 55.8 / 72.1 / 160.
LpPlan lp_plan(int dtype, int64_t rows, int64_t vocab, int top) {
    const int64_t per_load = dtype == QMM_F32 ? 4 : 8, loads = (vocab + 2 * per_load - 2) / per_load;  // (of the worst alignment)
    const int64_t fewest = (loads + 4 * kLpRuns - 1) / (4 * kLpRuns), enough = (compute_units() + rows / 2) / rows, most = loads < 4 * kLpStep ? 1 : std::min<int64_t>(64, loads / kLpThreads);
    int64_t parts = std::max(fewest, std::min(enough, most));
    const int64_t per = ((loads + parts - 1) / parts + 3) / 4 * 4;
    parts = (loads + per - 1) / per;
    return {(int)per, (int)parts};
}

template <typename T>
hipError_t run_logprobs(const T* logits, const LpPlan& p, int64_t stride, int64_t rows, int64_t vocab, const LpOut& out, void* workspace, hipStream_t s) {
    uint64_t* const keys = (uint64_t*)workspace;
    LpState* const states = (LpState*)(keys + rows * p.parts * out.top);
    const size_t lds = out.top > 0 ? (size_t)((p.per + 3) / 4) * 4 : 0;
    logprobs_kernel<T><<<dim3((unsigned)rows, (unsigned)p.parts), dim3(kLpThreads), lds, s>>>(logits, stride, (int)vocab, p.per, p.parts, states, keys, out);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.parts == 1) return e;
    if (p.parts <= 8) logprobs_join_kernel<T, 1><<<dim3((unsigned)rows), dim3(64), 0, s>>>(logits, stride, (int)vocab, p.parts, states, keys, out);
    else logprobs_join_kernel<T, 8><<<dim3((unsigned)rows), dim3(512), 0, s>>>(logits, stride, (int)vocab, p.parts, states, keys, out);
    return hipGetLastError();
}

}  // namespace

int64_t logprobs_workspace_bytes(int dtype, int64_t rows, int64_t vocab, int top) {
    rows = std::min(rows, kLpRows);
    const LpPlan p = lp_plan(dtype, rows, vocab, top);
    return p.parts == 1 ? 0 : rows * p.parts * ((int64_t)sizeof(LpState) + 8 * (int64_t)top);
}

hipError_t launch_logprobs(const void* logits, int dtype, int64_t stride, int64_t rows, int64_t vocab, const void* tokens, bool wide, int per_row, int top, float* chosen,
                           float* entropy, int32_t* top_ids, float* top_values, void* workspace, hipStream_t s) {
    const LpPlan p = lp_plan(dtype, std::min(rows, kLpRows), vocab, top);
    for (int64_t r0 = 0; r0 < rows; r0 += kLpRows) {
        const int64_t n = std::min(rows - r0, kLpRows);
        const LpOut out{tokens ? (const char*)tokens + r0 * per_row * (wide ? 8 : 4) : nullptr, wide, per_row, chosen ? chosen + r0 * per_row : nullptr, entropy + r0, top ? top_values + r0 * top : nullptr,
                        top ? top_ids + r0 * top : nullptr, top};
        const hipError_t e = dtype == QMM_F32 ? run_logprobs((const float*)logits + r0 * stride, p, stride, n, vocab, out, workspace, s)
                                              : run_logprobs((const uint16_t*)logits + r0 * stride, p, stride, n, vocab, out, workspace, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace qmm
