// Logits of a policy over tokens: penalties, biases, masks, temperature (trl_process_logits_*), and the log-probability and
// entropy of the stored tokens under them (trl_token_log_prob_*).  include/trl_value.h has the formulas.
//
// One element costs 2-4 bytes each way and a dozen instructions, so every kernel is one pass over the logits and bound by HBM as
// long as the vector units keep up (about 14 full-rate slots an element at 16 bits; v_exp_f32 takes four of them).
//   unit     A wave owns kSub consecutive tokens of the vocabulary and a run of rows of one sequence.  It never waits for another
//            wave after the prologue: no barrier, no LDS exchange inside a row; the softmax partials of a row ({max, sum, weighted
//            sum} a wave) are joined by a second, small launch, where there is more than one.
//   history  How often each token was seen lives in LDS, 4 bytes a token of the block's slice, bit 31 = seen in the prompt.  A
//            block scans the first row's history once; the next row of a rollout adds the one token that came since (a wave keeps a
//            64-token window of the history in registers).  Integer counts: the order of the atomics cannot change a result.
//   masks    A lane's 8 mask bits of the NEXT row are fetched a row ahead, so lanes with nothing allowed skip their logits without
//            a dependent load; masked logits are never read, whatever they hold.
//   softmax  In base 2 with one fma an element: d = z * c - M, e = 2^d, c = log2(e) / temperature (z before the division), all
//            relative to M = max * c as rounded, so that M's rounding cancels between the numerator and the sum.  It has to stay small
//            in the exponent for that, so rows with a maximum of 2^20 or more in magnitude (rows of the type's lowest value among
//            them) subtract first: d = (z - max) * c.  Everything is held in 32 bits.
// Measured at 8192 x 131072 bf16 (2.15 GB of logits; a large copy reaches 4.75 TB/s here, reading alone 3.7), us:
// (of 10 rows the mask leaves 4 whole, allows 3 every second token and 3 one in a hundred)
//                                    nothing on   a mask   a history of 1024   both and a bias
//   log-probability and entropy         464         416            574               514         4.6 TB/s, 3.7 with a history
//   their gradient                      871         810            880               800         4.9 TB/s
//   processed logits                    863         772            857               768         5.0 TB/s
// HBM bounds all but the first row's two columns with a history: there the vector units do, with the repeated places' factors beside the
// softmax.  One decoding step of 256 x 131072 with 4096 tokens of history takes 35 us (4.2 TB/s; reading and counting 4 MB of history 32
// times, once a slice, is what it has beside its 147 MB), one of 8 x 32000 7 us (the history's latency, then the row's).
#include "token_common.h"
#include "vec8.h"

namespace {

constexpr int kRowVecs = 4;                  // vectors of a lane in a row
constexpr int kBlk = kVec * kWave;           // 512 tokens: one vector of every lane
constexpr int kSub = kBlk * kRowVecs;        // 2048 tokens of a wave
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kFloor = -1.0e4f;            // 2^kFloor is 0: keeps 0 * (-inf) out of the entropy
constexpr u32 kSeenInPrompt = 0x80000000u;
typedef unsigned long long u64;

enum Mode { kProcess, kProcessBwd, kLogProb, kLogProbBwd };

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

__device__ __forceinline__ i64 load_int(const void *p, int wide, i64 i) { return wide ? ((const i64 *)p)[i] : (i64)((const int *)p)[i]; }

// ---- the block's counts --------------------------------------------------------------------------------------------------------
// token `off` of a sub-slice -> word: a lane's 8 tokens are two 16-byte pieces, each contiguous over the lanes (no bank conflict)
__device__ __forceinline__ int count_word(int off) {
    const int w = off & (kBlk - 1);
    return (off & ~(kBlk - 1)) + ((w & 4) << 6) + ((w >> 3) << 2) + (w & 3);
}

__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ void count_token(u32 *counts, i64 tok, i64 lo, int n, bool prompt) {
    const i64 off = tok - lo;
    if (off < 0 || off >= n) return;  // another slice's token, or no token at all (padding)
    u32 *c = counts + ((int)off & ~(kSub - 1)) + count_word((int)off & (kSub - 1));
    if (prompt) atomicOr(c, kSeenInPrompt);
    else atomicAdd(c, 1u);
}

// ---- a lane's share of a row: 8 tokens at `off` of the wave's sub-slice, of which the first n exist (n >= 8: all) -----------------------
__device__ __forceinline__ u32 mask_bits(int kind, const u8 *mask_lo, int off, int n) {
    if (n <= 0) return 0u;
    const u32 in = n >= kVec ? 0xffu : (1u << n) - 1u;
    if (kind == TRL_MASK_NONE) return in;
    if (kind == TRL_MASK_BITS) return mask_lo[off >> 3] & in;
    u32 bits = 0;
    if (n >= kVec) {
        typedef u32 u32x2 __attribute__((ext_vector_type(2)));
        typedef u32x2 u32x2_any __attribute__((aligned(1)));
        const u32x2 w = *(const u32x2_any *)(mask_lo + off);  // 8 truth values of one byte
        // Any byte but 0 allows (a byte tensor may be viewed as truth values): bit 7 of a byte is set where the rest or itself is not 0; the product
        // takes byte i's to bit 28 + i.  No carries in either.
        auto four = [](u32 x) { return (((((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u) * 0x00204081u) >> 28; };
        bits = four(w[0]) | four(w[1]) << 4;
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (i < n && mask_lo[off + i]) bits |= 1u << i;
    }
    return bits;
}

__device__ __forceinline__ void load_bias8(int kind, const char *bias_row, i64 tok, int n, float *b) {
    if (kind == kBiasF32) {
        Raw8<float> r{};
        load8((const float *)bias_row + tok, n, r);
        unpack8(r, b);
    } else if (kind == kBiasBf16) {
        Raw8<__bf16> r{};
        load8((const __bf16 *)bias_row + tok, n, r);
        unpack8(r, b);
    } else {
        Raw8<_Float16> r{};
        load8((const _Float16 *)bias_row + tok, n, r);
        unpack8(r, b);
    }
}

struct Penalties { float rep, inv_rep, pres, freq; bool subtracts; };

// keeps a rarely taken scalar branch one (8 selects in its place cost more than the row's softmax)
__device__ __forceinline__ void stay_branch(float &x) { asm volatile("" : "+v"(x)); }

// 8 counts of a lane.  `places`, the same in all lanes: bit i where any lane's count i is not 0 -- a wave looks at those alone.
struct Counts8 {
    u32 c[kVec], places;
    __device__ __forceinline__ Counts8() : places(0) {}
    __device__ __forceinline__ Counts8(const u32 *counts8, u32 p) : places(p) {
        if (!places) return;
        const u32x4 lo = *(const u32x4 *)counts8, hi = *(const u32x4 *)(counts8 + kBlk / 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) { c[i] = lo[i]; c[4 + i] = hi[i]; }
    }
    __device__ __forceinline__ bool any() const { return ((c[0] | c[1] | c[2]) | (c[3] | c[4] | c[5]) | (c[6] | c[7])) != 0; }
    __device__ __forceinline__ static float factor(float z, u32 c, const Penalties &p) {
        const float f = z > 0.0f ? p.inv_rep : p.rep;
        return c ? f : 1.0f;
    }
    __device__ __forceinline__ void apply(float *z, const Penalties &p) const {
        if (!places) return;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            if (places & (1u << i)) {
                z[i] *= factor(z[i], c[i], p);
                stay_branch(z[i]);
                if (p.subtracts) {
                    const u32 k = c[i] & ~kSeenInPrompt;
                    z[i] -= k ? fmaf((float)k, p.freq, p.pres) : 0.0f;
                }
            }
        }
    }
    __device__ __forceinline__ void slope(float *d, const float *raw, const Penalties &p) const {
        if (!places) return;
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (places & (1u << i)) {
                d[i] *= factor(raw[i], c[i], p);
                stay_branch(d[i]);
            }
    }
};

// z where bit i allows it, else `other`: two instructions a place
__device__ __forceinline__ float where_allowed(u32 bits, int i, float z, u32 other) {
    const int m = __builtin_amdgcn_sbfe((int)bits, i, 1);  // all bits set where it is allowed
    float r;
    asm("v_bfi_b32 %0, %1, %2, %3" : "=v"(r) : "v"(m), "v"(z), "v"(other));
    return r;
}
constexpr u32 kNegInfBits = 0xff800000u;
// What stands for -inf in masked places of the log-probability's forward pass: 0 * d stays finite there without a clamp.  Waves whose
// maximum comes near it, and waves whose weighted sum is NaN (infinities in allowed places), start over with -inf and a clamp.  So do
// all waves at a scale of up to 1e-23 (temperatures from 1.4e23 on): it has to be far below in the exponent, where it stands at -1e7
// at that scale, ten times the 2^20 that a shift may add.
constexpr float kFarBelow = -1e30f, kLeastScale = 1e-23f;

// (the builtin would first pass values of unknown origin through a multiplication by one)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// the shift of d = z * c - shift for a row's (or a wave's) largest value m; *steep: d = (z - m) * c, see the head of the file
__device__ __forceinline__ float softmax_shift(float m, float c, bool *steep) {
    const float m2 = m * c;
    *steep = fabsf(m2) >= 0x1p20f && !__builtin_isinf(m);
    return m == neg_inf() || *steep ? 0.0f : m2;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// A kernel argument as a scalar of its own.  Arguments are fetched 16 words at a time, and one that has to leave the scalar registers
// would take its 15 neighbours with it, to vector lanes and back in every row.
__device__ __forceinline__ int scalar(int v) {
    v = __builtin_amdgcn_readfirstlane(v);
    asm volatile("" : "+s"(v));
    return v;
}
__device__ __forceinline__ i64 scalar(i64 v) { return (i64)((u64)(u32)scalar((int)v) | (u64)(u32)scalar((int)(v >> 32)) << 32); }
__device__ __forceinline__ i64 scalar(int64_t v) { return scalar((i64)v); }
template <typename P>
__device__ __forceinline__ P *scalar(P *p) { return (P *)scalar((i64)p); }

// the same value, as far as the compiler knows a new one
__device__ __forceinline__ int again(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// What a lane knows of row t0 + lane before the block's rows begin: a row's scalars are then one v_readlane away, not a memory latency.
struct RowAhead {
    int want = 0;    // PEN: length of the history
    int action = 0;  // -1: padding; 0x7fffffff: no token of the vocabulary
    // backward: d raw = -e (ca + cb d), + g at the action
    float shift = 0.0f, top = 0.0f, ca = 0.0f, cb = 0.0f, g = 0.0f;
    int kind = 0;  // kRowZero, kRowSteep, kRowCold
};
// no gradient; subtract first; 1 / temperature comes last (in the coefficients it may overflow, and what has no weight would be 0 * infinity)
enum { kRowZero = 1, kRowSteep = 2, kRowCold = 4 };
constexpr float kColdest = 0x1p64f;  // 1 / temperature in the coefficients up to here: 2^63 is left for the gradients, kFloor and the sums

// The results of a row from its largest value, the sum and the weighted sum relative to it.
__device__ __forceinline__ void finish_row(const TokenArgs &a, i64 r, i64 y, float m, float s, float u, float scale, float z_action) {
    float log_prob = 0.0f, entropy = 0.0f, log2s = 0.0f;
    if (y < 0) {
        m = neg_inf();
    } else {
        bool steep;
        const float shift = softmax_shift(m, scale, &steep);
        if (m == neg_inf() && s == 0.0f) {  // nothing allowed, or nothing possible
            log_prob = neg_inf();
        } else {
            const float z = steep ? z_action - m : z_action;
            log2s = log2f(s);
            entropy = kLn2 * (log2s - u / s);
            log_prob = kLn2 * (fmaf(z, scale, -shift) - log2s);
        }
        if (y >= a.V) log_prob = __builtin_nanf("");
    }
    a.log_prob[r] = log_prob;
    if (a.entropy) a.entropy[r] = entropy;
    if (a.stats) { a.stats[2 * r] = m; a.stats[2 * r + 1] = log2s; }
}

// Joins a row's partials (one a sub-slice): called by a whole wave, or by one lane for itself.
template <bool WAVE>
__device__ __forceinline__ void join_row(const TokenArgs &a, i64 r, i64 y, const float4 *part, i64 nsubs, float z_action) {
    const int lane = WAVE ? threadIdx.x & (kWave - 1) : 0;
    constexpr int kStep = WAVE ? kWave : 1;
    float m = neg_inf(), s = 0.0f, u = 0.0f, scale = 0.0f;
    if (y >= 0) {
        for (i64 i = lane; i < nsubs; i += kStep) m = fmaxf(m, part[i].x);
        if (WAVE) m = wave_max(m);
        scale = kLog2e * (1.0f / (a.temp_t ? a.temp_t[r / a.T] : a.temp));  // the row kernel's own bits
        bool steep;
        const float shift = softmax_shift(m, scale, &steep);
        for (i64 i = lane; i < nsubs; i += kStep) {
            const float4 q = part[i];
            float d = 0.0f;
            if (q.x != m) {
                bool own;  // whether the wave's values are relative to q.x itself
                const float its = softmax_shift(q.x, scale, &own);
                if (q.x == neg_inf()) d = neg_inf();
                else if (own) d = steep ? (q.x - m) * scale : fmaf(q.x, scale, -shift);
                else d = steep ? fmaf(-m, scale, its) : its - shift;
            }
            const float w = exp2_hw(d);
            s = fmaf(w, q.y, s);
            u = fmaf(w, fmaf(q.y, fmaxf(d, kFloor), q.z), u);
        }
        if (WAVE) {
            s = wave_sum(s);
            u = wave_sum(u);
        }
    }
    if (lane == 0) finish_row(a, r, y, m, s, u, scale, z_action);
}

// fp32 log-probabilities under penalties and a bias hold more than the 128 registers of four waves a SIMD: three, in blocks that fill them
// (8192 x 131072 with a mask: 711 us, in blocks of 12 waves 734, of 8 837; four waves with 142 registers spilled 1090).
template <typename T, int MODE, bool PEN, bool BIAS> constexpr bool kHeavy = MODE == kLogProb && PEN && BIAS && sizeof(T) == 4;
// waves of a block: the launch picks up to that many
template <typename T, int MODE, bool PEN, bool BIAS> constexpr int kMostWaves = PEN && !kHeavy<T, MODE, PEN, BIAS> ? 16 : 4;
template <typename T, int MODE, bool PEN, bool BIAS> constexpr int kSimdWaves = kHeavy<T, MODE, PEN, BIAS> ? 3 : 4;

template <typename T, int MODE, bool PEN, bool BIAS>
__global__ __launch_bounds__((kMostWaves<T, MODE, PEN, BIAS>) * kWave, (kSimdWaves<T, MODE, PEN, BIAS>)) void token_kernel(TokenArgs a) {
    extern __shared__ __align__(16) u32 lds_counts[];  // PEN: a sub-slice a wave
    const int W = blockDim.x / kWave;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const u32 nslices = (u32)a.nslices, nchunks = (u32)a.nchunks, rest = scalar((int)(blockIdx.x / nslices)), slice = blockIdx.x - rest * nslices;
    const i64 b = scalar((int)(rest / nchunks)), t0 = (i64)(rest - (u32)b * nchunks) * a.chunk;
    const int rows = a.T - t0 < a.chunk ? (int)(a.T - t0) : (int)a.chunk;
    const i64 slice_lo = (i64)slice * W * kSub, lo = slice_lo + wave * kSub, r0 = b * a.T + t0;
    u32 *counts = lds_counts + wave * kSub;

    RowAhead mine;
    if (lane < rows) {
        if constexpr (PEN) {
            const i64 n = a.lengths ? load_int(a.lengths, a.lengths_wide, r0 + lane) : a.L;
            mine.want = n < 0 ? 0 : n > a.L ? (int)a.L : (int)n;
        }
        if constexpr (MODE == kLogProb || MODE == kLogProbBwd) {
            const i64 y = load_int(a.action, a.action_wide, r0 + lane);
            mine.action = y < 0 ? -1 : y >= a.V ? 0x7fffffff : (int)y;
        }
    }
    int h = 0, prompt = 0;  // history tokens that the counts hold; where the generated ones begin
    if constexpr (PEN) {
        const i64 p = a.prompt ? load_int(a.prompt, a.prompt_wide, b) : 0;
        prompt = p < 0 ? 0 : p > a.L ? (int)a.L : (int)p;
        // four tokens a thread at a time; the first are on their way before the history's length is known
        constexpr int kAhead = 4;
        i64 ahead[kAhead];
        auto fetch = [&](int from, int end) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int j = from + i * (int)blockDim.x + (int)threadIdx.x;
                ahead[i] = j < end ? load_int(a.tokens, a.tokens_wide, b * a.tokens_sb + j) : -1;
            }
        };
        fetch(0, (int)a.L < kAhead * (int)blockDim.x ? (int)a.L : kAhead * (int)blockDim.x);
        u32x4 *c4 = (u32x4 *)lds_counts;
#pragma unroll
        for (int i = 0; i < kSub / 4 / kWave; ++i) c4[threadIdx.x + i * blockDim.x] = u32x4{0, 0, 0, 0};
        __syncthreads();
        h = read_lane(mine.want, 0);
        for (int from = 0; from < h; from += kAhead * (int)blockDim.x) {
            if (from) fetch(from, h);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int j = from + i * (int)blockDim.x + (int)threadIdx.x;
                if (j < h) count_token(lds_counts, ahead[i], slice_lo, W * kSub, j < prompt);
            }
        }
        __syncthreads();
    }
    if (lo >= a.V) return;

    Penalties pen{a.rep_t ? a.rep_t[b] : a.rep, 0.0f, a.pres_t ? a.pres_t[b] : a.pres, a.freq_t ? a.freq_t[b] : a.freq, false};
    pen.inv_rep = 1.0f / pen.rep;
    pen.subtracts = pen.pres != 0.0f || pen.freq != 0.0f;
    const float inv_temp = 1.0f / (a.temp_t ? a.temp_t[b] : a.temp);
    const float scale = kLog2e * inv_temp;
    const bool needs_z = MODE != kProcessBwd || (PEN && (a.rep_t || a.rep != 1.0f));
    if constexpr (MODE == kLogProbBwd) {
        if (lane < rows) {
            const i64 r = r0 + lane;
            const float m = a.stats[2 * r], log2s = a.stats[2 * r + 1];
            if (mine.action < 0 || (m == neg_inf() && log2s == 0.0f)) {  // padding, or nothing allowed (a row of NaN has a NaN in its sum)
                mine.kind = kRowZero;
            } else {
                bool steep;
                mine.shift = softmax_shift(m, scale, &steep);
                mine.top = m;
                const float g_h = a.g_entropy ? a.g_entropy[r] : 0.0f, rs = exp2_hw(-log2s);
                float g = a.g_log_prob ? a.g_log_prob[r] : 0.0f;
                if (mine.action == 0x7fffffff) g = __builtin_nanf("");
                const float entropy = a.g_entropy ? a.entropy[r] : 0.0f;
                const bool cold = inv_temp > kColdest;
                const float f = cold ? 1.0f : inv_temp;
                mine.ca = rs * (g + g_h * (entropy - kLn2 * log2s)) * f;
                mine.cb = rs * g_h * kLn2 * f;
                mine.g = g * f;
                mine.kind = (steep ? kRowSteep : 0) | (cold ? kRowCold : 0);
            }
        }
    }

    // bit k * 8 + i: some token of place i of the wave's vector k was seen
    u32 seen_places = 0;
    if constexpr (PEN) {
#pragma unroll
        for (int k = 0; k < kRowVecs; ++k) {
            const Counts8 c(counts + k * kBlk + lane * 4, 1);
#pragma unroll
            for (int i = 0; i < kVec; ++i) seen_places |= __any(c.c[i] != 0) ? 1u << (k * kVec + i) : 0u;
        }
    }
    // a window of the history, a token a lane, as its place in the sub-slice (negative: elsewhere), and which of them are here at all
    const char *tokens = PEN ? scalar((const char *)a.tokens + b * a.tokens_sb * (a.tokens_wide ? 8 : 4)) : nullptr;
    const int tokens_wide = PEN ? scalar(a.tokens_wide) : 0, n_tokens = PEN ? scalar((int)a.L) : 0;
    int win_lo = 0, win_end = 0, win = -1;
    unsigned long long win_hits = 0;
    auto grow_history = [&](int want) {
        if (want < h) {  // not a rollout's order: count anew
            wave_fence();
            u32x4 *c4 = (u32x4 *)counts;
#pragma unroll
            for (int i = 0; i < kSub / 4 / kWave; ++i) c4[lane + i * kWave] = u32x4{0, 0, 0, 0};
            wave_fence();
            h = 0;
            seen_places = 0;
        }
        while (h < want) {
            if (h < win_lo || h >= win_end) {
                win_lo = h;
                win_end = h + kWave;
                const i64 at = h + lane < n_tokens ? load_int(tokens, tokens_wide, h + lane) - lo : -1;
                win = at >= 0 && at < kSub ? (int)at : -1;
                win_hits = __ballot(win >= 0);
            }
            const int end = want < win_end ? want : win_end;
            unsigned long long todo = win_hits >> (h - win_lo);
            if (end - h < kWave) todo &= (1ull << (end - h)) - 1;
            if (todo) {
                wave_fence();
                for (; todo; todo &= todo - 1) {
                    const int j = h + __builtin_ctzll(todo), at = read_lane(win, j - win_lo);
                    if (lane == 0) count_token(counts, at, 0, kSub, j < prompt);
                    seen_places |= 1u << (at / kBlk * kVec + at % kVec);
                }
                wave_fence();
            }
            h = end;
        }
    };

    const float least_max = scale > kLeastScale ? 0.01f * kFarBelow : __builtin_inff();  // above it, masked places may hold kFarBelow
    const i64 left = a.V - lo;
    const int mask_kind = scalar(a.mask_kind);
    const i64 logits_st = scalar(a.logits_st), out_st = scalar(a.out_st), mask_st = scalar(a.mask_st), nsubs = scalar(a.nsubs);
    // of the next row
    const T *z_next = scalar((const T *)a.logits + b * a.logits_sb + t0 * a.logits_st + lo);
    const T *g_next = scalar((const T *)a.grad_out + r0 * a.V + lo);
    T *out_next = scalar((T *)a.out + b * a.out_sb + t0 * a.out_st + lo);
    const u8 *mask_next = scalar((const u8 *)a.mask + b * a.mask_sb + t0 * a.mask_st + (mask_kind == TRL_MASK_BITS ? lo >> 3 : lo));
    const int bias_kind = scalar(a.bias_kind);
    const i64 bias_st = scalar(a.bias_st), vocabulary = scalar(a.V);
    const char *bias_next = scalar((const char *)a.bias + b * a.bias_sb + t0 * a.bias_st);
    float4 *part_next = scalar((float4 *)a.partials + r0 * a.nsubs + lo / kSub);
    float *z_action = scalar(a.z_action + r0);

    const int lane0 = lane;
    const bool alone = nsubs == 1;  // a row is one wave's: no joining launch, lane i keeps row i's numbers
    float own_m = neg_inf(), own_s = 0.0f, own_u = 0.0f, own_z = neg_inf();
    // FULL: every token of the sub-slice exists
    auto run_rows = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        int off[kRowVecs], nv[kRowVecs];
        u32 next_bits[kRowVecs];
#pragma unroll
        for (int k = 0; k < kRowVecs; ++k) {
            off[k] = k * kBlk + lane0 * kVec;
            nv[k] = FULL || left - off[k] > kVec ? kVec : left < off[k] ? 0 : (int)(left - off[k]);
            next_bits[k] = mask_bits(mask_kind, mask_next, off[k], nv[k]);
        }
        float bias[BIAS ? kRowVecs : 1][kVec];
        if constexpr (BIAS) {
            if (bias_st == 0) {  // one bias for all rows of the block: kept in registers
#pragma unroll
                for (int k = 0; k < kRowVecs; ++k) load_bias8(bias_kind, bias_next, lo + off[k], nv[k], bias[k]);
            }
        }
        for (int i_row = 0; i_row < rows; ++i_row) {
            const int lane = again(lane0);  // what follows from it is cheaper to compute in each row than to keep
#pragma unroll
            for (int k = 0; k < kRowVecs; ++k) {
                off[k] = k * kBlk + lane * kVec;
                nv[k] = FULL || left - off[k] > kVec ? kVec : left < off[k] ? 0 : (int)(left - off[k]);
            }
            u32 bits[kRowVecs];
            bool live[kRowVecs];  // of the wave
#pragma unroll
            for (int k = 0; k < kRowVecs; ++k) {
                bits[k] = next_bits[k];
                live[k] = __any(bits[k] != 0);
            }
            if (mask_st != 0 && i_row + 1 < rows) {
                mask_next += mask_st;
#pragma unroll
                for (int k = 0; k < kRowVecs; ++k) next_bits[k] = mask_bits(mask_kind, mask_next, off[k], nv[k]);
            }
            const T *z_row = z_next, *g_row = g_next;
            T *out_row = out_next;
            const char *bias_row = bias_next;
            float4 *part = part_next;
            z_next += logits_st;
            out_next += out_st;
            bias_next += bias_st;
            part_next += nsubs;
            if constexpr (MODE == kProcessBwd) g_next += vocabulary;
            const int y = MODE == kLogProb || MODE == kLogProbBwd ? read_lane(mine.action, i_row) : 0;
            const int kind = MODE == kLogProbBwd ? read_lane(mine.kind, i_row) : 0;
            if (MODE == kLogProb && y < 0) continue;  // padding: the joining launch answers for it
            if (MODE == kLogProbBwd && (kind & kRowZero)) {
                const float zero[kVec] = {};
#pragma unroll
                for (int k = 0; k < kRowVecs; ++k)
                    if (FULL || nv[k] > 0) store8(out_row + off[k], nv[k], zero);
                continue;
            }
            // -- loads; a lane with nothing allowed makes none
            Raw8<T> zr[kRowVecs], gr[MODE == kProcessBwd ? kRowVecs : 1];
#pragma unroll
            for (int k = 0; k < kRowVecs; ++k) {
                zr[k] = Raw8<T>{};
                if (MODE != kProcessBwd && bits[k]) load8(z_row + off[k], nv[k], zr[k]);
                if constexpr (MODE == kProcessBwd) {
                    gr[k] = Raw8<T>{};
                    if (bits[k]) load8(g_row + off[k], nv[k], gr[k]);
                }
            }
            if constexpr (PEN) {
                const int want = read_lane(mine.want, i_row);
                if (want != h) grow_history(want);
            }
            if constexpr (BIAS) {
                if (bias_st != 0) {
#pragma unroll
                    for (int k = 0; k < kRowVecs; ++k) load_bias8(bias_kind, bias_row, lo + off[k], nv[k], bias[k]);
                }
            }
            // before the temperature
            auto processed = [&](int k, float *z, const Counts8 &c, u32 fill) {
                if constexpr (PEN) c.apply(z, pen);
                if constexpr (BIAS) {
#pragma unroll
                    for (int i = 0; i < kVec; ++i) z[i] += bias[k][i];
                }
                if constexpr (MODE == kProcess) {
#pragma unroll
                    for (int i = 0; i < kVec; ++i) z[i] *= inv_temp;
                }
                if (!FULL || !__all(bits[k] == 0xffu)) {
#pragma unroll
                    for (int i = 0; i < kVec; ++i) z[i] = where_allowed(bits[k], i, z[i], fill);
                }
            };
            const u32 *counts8 = counts + lane * 4;

            if constexpr (MODE == kLogProb) {
                float z[kRowVecs][kVec];
                float m = neg_inf(), z_y = neg_inf();
                const i64 at = y - lo;
#pragma unroll
                for (int k = 0; k < kRowVecs; ++k) {
                    if (!live[k]) continue;
                    unpack8(zr[k], z[k]);
                    processed(k, z[k], PEN ? Counts8(counts8 + k * kBlk, seen_places >> (k * kVec) & 0xffu) : Counts8(), __builtin_bit_cast(u32, kFarBelow));
#pragma unroll
                    for (int i = 0; i < kVec; i += 2) m = max3(m, z[k][i], z[k][i + 1]);
                    if (at >= k * kBlk && at < (k + 1) * kBlk) {  // one vector of one wave
                        float mine_z = neg_inf();
#pragma unroll
                        for (int i = 0; i < kVec; ++i)
                            if (((int)at & (kVec - 1)) == i) mine_z = bits[k] & (1u << i) ? z[k][i] : neg_inf();
                        z_y = read_lane(mine_z, ((int)at & (kBlk - 1)) / kVec);
                    }
                }
                m = wave_max(m);
                float s = 0.0f, u = 0.0f;
                bool steep;
                float shift = softmax_shift(m, scale, &steep);
                bool careful = steep || !(m > least_max);  // (not live at all among them)
                if (!careful) {
#pragma unroll
                    for (int k = 0; k < kRowVecs; ++k) {
                        if (!live[k]) continue;
#pragma unroll
                        for (int i = 0; i < kVec; ++i) {
                            const float d = fmaf(z[k][i], scale, -shift), e = exp2_hw(d);
                            s += e;
                            u = fmaf(e, d, u);
                        }
                    }
                    s = wave_sum(s);
                    u = wave_sum(u);
                    careful = __builtin_isnan(u) && !__builtin_isnan(s);
                }
                if (careful) {
                    m = neg_inf();
                    s = u = 0.0f;
#pragma unroll
                    for (int k = 0; k < kRowVecs; ++k) {
                        if (!live[k]) continue;
#pragma unroll
                        for (int i = 0; i < kVec; ++i) {
                            z[k][i] = where_allowed(bits[k], i, z[k][i], kNegInfBits);
                            m = fmaxf(m, z[k][i]);
                        }
                    }
                    m = wave_max(m);
                    shift = softmax_shift(m, scale, &steep);
#pragma unroll
                    for (int k = 0; k < kRowVecs; ++k) {
                        if (!live[k]) continue;
#pragma unroll
                        for (int i = 0; i < kVec; ++i) {
                            const float d = fmaf(steep ? z[k][i] - m : z[k][i], scale, -shift), e = exp2_hw(d);
                            s += e;
                            u = fmaf(e, fmaxf(d, kFloor), u);
                        }
                    }
                    s = wave_sum(s);
                    u = wave_sum(u);
                }
                if (alone) {
                    const bool its = lane == i_row;
                    own_m = its ? m : own_m;
                    own_s = its ? s : own_s;
                    own_u = its ? u : own_u;
                    own_z = its ? z_y : own_z;
                } else if (lane == 0) {
                    *part = make_float4(m, s, u, 0.0f);
                    if (at >= 0 && at < kSub) z_action[i_row] = z_y;
                }
            } else {
                const float shift = read_lane(mine.shift, i_row), top = read_lane(mine.top, i_row), ca = read_lane(mine.ca, i_row),
                            cb = read_lane(mine.cb, i_row), g = read_lane(mine.g, i_row);
#pragma unroll
                for (int k = 0; k < kRowVecs; ++k) {
                    float z[kVec];
                    if (!live[k]) {
#pragma unroll
                        for (int i = 0; i < kVec; ++i) z[i] = MODE == kProcess ? neg_inf() : 0.0f;
                    } else {
                        const Counts8 c = PEN ? Counts8(counts8 + k * kBlk, seen_places >> (k * kVec) & 0xffu) : Counts8();
                        if constexpr (MODE == kProcessBwd && PEN) {  // the sign of a logit matters where it was repeated, and nowhere else
                            if (needs_z && c.places && bits[k] && c.any()) load8(z_row + off[k], nv[k], zr[k]);
                        }
                        float raw[kVec];
                        unpack8(zr[k], raw);
                        if constexpr (MODE == kProcessBwd) {
                            unpack8(gr[k], z);
#pragma unroll
                            for (int i = 0; i < kVec; ++i) z[i] *= inv_temp;
                        } else {
#pragma unroll
                            for (int i = 0; i < kVec; ++i) z[i] = raw[i];
                            processed(k, z, c, kNegInfBits);
                        }
                        if constexpr (MODE == kLogProbBwd) {
                            if (kind & kRowSteep) {
#pragma unroll
                                for (int i = 0; i < kVec; ++i) z[i] -= top;
                            }
#pragma unroll
                            for (int i = 0; i < kVec; ++i) {
                                const float d = fmaf(z[i], scale, -shift), e = exp2_hw(d);
                                z[i] = -e * fmaf(cb, fmaxf(d, kFloor), ca);
                            }
                            const i64 at = y - lo - k * kBlk;
                            if (at >= 0 && at < kBlk) {  // one vector of one wave
#pragma unroll
                                for (int i = 0; i < kVec; ++i)
                                    if (lane * kVec + i == (int)at) z[i] += g;
                            }
                            if (kind & kRowCold) {
#pragma unroll
                                for (int i = 0; i < kVec; ++i) z[i] *= inv_temp;
                            }
                        }
                        if constexpr (PEN && MODE != kProcess) c.slope(z, raw, pen);
                        // masked places have e = 0; an action among them, and coefficients that are no numbers, need the zero itself
                        if (MODE == kProcessBwd || MODE == kLogProbBwd) {
                            if (!__all(bits[k] == 0xffu)) {
#pragma unroll
                                for (int i = 0; i < kVec; ++i) z[i] = where_allowed(bits[k], i, z[i], 0u);
                            }
                        }
                    }
                    if (FULL || nv[k] > 0) store8(out_row + off[k], nv[k], z);
                }
            }
        }
    };
    if (left >= kSub) run_rows(Bool<true>());
    else run_rows(Bool<false>());
    if (MODE == kLogProb && alone && lane < rows) {
        const i64 y = mine.action == 0x7fffffff ? a.V : mine.action;
        finish_row(a, r0 + lane, y, own_m, own_s, own_u, scale, own_z);
    }
}

// A wave a row: 16 bytes a sub-slice to read, so a launch's latency bounds it (2.2 us for 4 rows, 5 us for 8192 of 64 sub-slices).  A lane a row
// where there are up to kSerialSubs (32768 rows of 2, 4 and 8: 4.2, 4.8 and 7.9 us, with a wave each 11, 13 and 15; of 16 11 and 14, but 64 rows
// of 16 6.5 and 4.0).  A last-block join inside the row kernel would save the launch but costs that kernel an atomic, a fence and registers a
// row; it measured slower.
constexpr i64 kSerialSubs = 8;
template <bool WAVE>
__global__ __launch_bounds__(256) void token_join_kernel(TokenArgs a) {
    const i64 r = WAVE ? (i64)blockIdx.x * 4 + threadIdx.x / kWave : (i64)blockIdx.x * 256 + threadIdx.x;
    if (r >= a.B * a.T) return;
    const i64 y = load_int(a.action, a.action_wide, r);
    join_row<WAVE>(a, r, y, (const float4 *)a.partials + r * a.nsubs, a.nsubs, y >= 0 && y < a.V ? a.z_action[r] : 0.0f);
}

template <typename P>
void advance(P *&p, i64 bytes) { if (p) p = (P *)((uintptr_t)p + (uintptr_t)bytes); }

// The n sequences from b0 on: rows of different sequences share nothing but strides.
TokenArgs sequences(const TokenArgs &a, i64 b0, i64 n) {
    TokenArgs p = a;
    auto width = [](int wide) -> i64 { return wide ? 8 : 4; };
    const i64 r0 = b0 * a.T, es = a.dtype == TRL_F32 ? 4 : 2;
    advance(p.logits, b0 * a.logits_sb * es);
    advance(p.out, b0 * a.out_sb * es);
    advance(p.grad_out, r0 * a.V * es);
    advance(p.tokens, b0 * a.tokens_sb * width(a.tokens_wide));
    advance(p.lengths, r0 * width(a.lengths_wide));
    advance(p.prompt, b0 * width(a.prompt_wide));
    advance(p.action, r0 * width(a.action_wide));
    advance(p.bias, b0 * a.bias_sb);
    advance(p.mask, b0 * a.mask_sb);
    for (const float **x : {&p.rep_t, &p.pres_t, &p.freq_t, &p.temp_t}) advance(*x, b0 * 4);
    for (float **x : {&p.log_prob, &p.entropy, &p.z_action}) advance(*x, r0 * 4);
    for (const float **x : {&p.g_log_prob, &p.g_entropy}) advance(*x, r0 * 4);
    advance(p.stats, r0 * 8);
    advance(p.partials, r0 * a.nsubs * 16);
    p.B = n;
    return p;
}

// Calls launch(args) on runs of sequences that one launch can take, `each` being the threads of one; 2 where a single sequence needs more.
template <typename F>
int in_launches(const TokenArgs &a, i64 each, F launch) {
    const i64 most = kMostThreads / each;
    if (most == 0) return 2;
    if (a.B <= most) {
        launch(a);
    } else {
        for (i64 b = 0; b < a.B; b += most) launch(sequences(a, b, a.B - b < most ? a.B - b : most));
    }
    return 0;
}

// Blocks of as many waves as an even split of the vocabulary gives them, up to 8 beside a history: two such blocks share a compute unit,
// and one streams while the other counts.  Up to 16, one block a unit, where the counting is shared by enough: long histories, or runs of
// many rows (16 waves and 8: 256 x 131072 bf16 with 4096 tokens 35 us and 37; 8192 x 131072 bf16 with every step on, backward, 800 and 852,
// forward 534 and 568; but 910 x 50263 fp32 with gradient 165 and 158).
template <typename T, int MODE, bool PEN, bool BIAS>
int launch_waves(hipStream_t s, TokenArgs &a) {
    a.nsubs = token_subs(a.V);
    const i64 rows = a.B * a.T;
    i64 most = kMostWaves<T, MODE, PEN, BIAS>;
    if (most > 8) {
        const i64 blocks = (a.nsubs + most - 1) / most * rows;
        if (blocks < 1024 || (a.L < 2048 && blocks < 4096)) most = 8;
    }
    a.nslices = (a.nsubs + most - 1) / most;
    const i64 waves = (a.nsubs + a.nslices - 1) / a.nslices;
    // The run of rows of a block (a lane holds a row's scalars): as few rounds of blocks as the chip takes at a time, counted in rows, with
    // the block's start as some rows more -- short runs count the history over and over, long ones leave a last round half empty.
    const i64 slots = 256 * (4 * kSimdWaves<T, MODE, PEN, BIAS> / waves);
    const double start = PEN ? 2.0 + (double)a.L / 1024.0 : 1.0;
    double best = 0.0;
    for (i64 c = 1; c <= kWave && c <= a.T; ++c) {
        const i64 blocks = a.nslices * a.B * ((a.T + c - 1) / c), rounds = (blocks + slots - 1) / slots;
        const double cost = (double)rounds * ((double)c + start);
        if (c == 1 || cost < best) { best = cost; a.chunk = c; }
    }
    a.nchunks = (a.T + a.chunk - 1) / a.chunk;
    const i64 threads = waves * kWave, blocks = a.nslices * a.nchunks;  // blocks of a sequence
    const size_t lds = (PEN ? waves * kSub * sizeof(u32) : 0);
    return in_launches(a, blocks * threads, [&](const TokenArgs &p) {
        hipLaunchKernelGGL((token_kernel<T, MODE, PEN, BIAS>), dim3((unsigned)(blocks * p.B)), dim3((unsigned)threads), lds, s, p);
    });
}
template <typename T, int MODE>
int launch_mode(hipStream_t s, TokenArgs &a) {
    if constexpr (MODE != kProcessBwd) {
        if (a.bias_kind != kBiasNone) return a.tokens ? launch_waves<T, MODE, true, true>(s, a) : launch_waves<T, MODE, false, true>(s, a);
    }
    return a.tokens ? launch_waves<T, MODE, true, false>(s, a) : launch_waves<T, MODE, false, false>(s, a);
}
template <int MODE>
int launch_dtype(hipStream_t s, TokenArgs &a) {
    switch (a.dtype) {
        case TRL_F32: return launch_mode<float, MODE>(s, a);
        case TRL_BF16: return launch_mode<__bf16, MODE>(s, a);
        default: return launch_mode<_Float16, MODE>(s, a);
    }
}

}  // namespace

i64 token_subs(i64 V) { return (V + kSub - 1) / kSub; }

int launch_process_logits(hipStream_t s, TokenArgs a) { return launch_dtype<kProcess>(s, a); }
int launch_process_logits_bwd(hipStream_t s, TokenArgs a) { return launch_dtype<kProcessBwd>(s, a); }
int launch_token_log_prob(hipStream_t s, TokenArgs a) {
    a.nsubs = token_subs(a.V);
    const bool wave = a.nsubs > kSerialSubs;
    const i64 joining = a.T * (wave ? kWave : 1);  // threads of a sequence
    if (a.nsubs > 1 && joining > kMostThreads) return 2;
    const int rc = launch_dtype<kLogProb>(s, a);
    if (rc || a.nsubs == 1) return rc;
    return in_launches(a, joining, [&](const TokenArgs &p) {
        const i64 rows = p.B * p.T;
        if (wave) hipLaunchKernelGGL(token_join_kernel<true>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, p);
        else hipLaunchKernelGGL(token_join_kernel<false>, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, s, p);
    });
}
int launch_token_log_prob_bwd(hipStream_t s, TokenArgs a) { return launch_dtype<kLogProbBwd>(s, a); }
