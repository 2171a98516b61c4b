// Logits of a policy over tokens: penalties, biases, masks, temperature (trl_process_logits_*), and the log-probability and
// entropy of the stored tokens under them (trl_token_log_prob_*).  include/trl_value.h has the formulas.
//
// One element costs 2-4 bytes each way and a dozen instructions, so every kernel is one pass over the logits and bound by HBM as
// long as the vector units keep up (about 14 full-rate slots an element at 16 bits; v_exp_f32 takes four of them).
//   unit     A wave owns kSub consecutive tokens of the vocabulary and a run of rows of one sequence.  It never waits for another
//            wave after the prologue: no barrier, no LDS exchange inside a row; the softmax partials of a row ({max, sum, weighted
//            sum} a wave) are joined by a second, small launch.
//   history  How often each token was seen lives in LDS, 4 bytes a token of the block's slice, bit 31 = seen in the prompt.  A
//            block scans the first row's history once; the next row of a rollout adds the one token that came since (a wave keeps a
//            64-token window of the history in registers).  Integer counts: the order of the atomics cannot change a result.
//   masks    A lane's 8 mask bits of the NEXT row are fetched a row ahead, so lanes with nothing allowed skip their logits without
//            a dependent load; masked logits are never read, whatever they hold.
//   softmax  In base 2 with one fma an element: d = z * log2(e) - M, e = 2^d, all relative to M = max * log2(e) as rounded, so that
//            M's rounding cancels between the numerator and the sum.  That rounding has to stay small in the exponent, so rows whose
//            maximum is 2^20 or more in magnitude (rows of the type's lowest value among them) subtract first: d = (z - max) * log2(e).
//            Everything is held in 32 bits.
#include "token_common.h"
#include "vec8.h"

namespace {

constexpr int kRowVecs = 4;                  // vectors of a lane in a row
constexpr int kBlk = kVec * kWave;           // 512 tokens: one vector of every lane
constexpr int kSub = kBlk * kRowVecs;        // 2048 tokens of a wave
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kFloor = -1.0e4f;            // 2^kFloor is 0: keeps 0 * (-inf) out of the entropy
constexpr u32 kSeenInPrompt = 0x80000000u;

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

__device__ __forceinline__ void count_token(u32 *counts, i64 tok, i64 lo, i64 n, bool prompt) {
    const i64 off = tok - lo;
    if (off < 0 || off >= n) return;  // another slice's token, or no token at all (padding)
    u32 *c = counts + (off & ~(i64)(kSub - 1)) + count_word((int)(off & (kSub - 1)));
    if (prompt) atomicOr(c, kSeenInPrompt);
    else atomicAdd(c, 1u);
}

// ---- one row's share of a lane -------------------------------------------------------------------------------------------------
__device__ __forceinline__ u32 mask_bits(const TokenArgs &a, const u8 *mask_row, i64 tok, int n) {
    if (n <= 0) return 0u;
    const u32 in = n >= kVec ? 0xffu : (1u << n) - 1u;
    if (a.mask_kind == TRL_MASK_NONE) return in;
    if (a.mask_kind == TRL_MASK_BITS) return mask_row[tok >> 3] & in;  // tok is a multiple of 8
    u32 bits = 0;
    if (n >= kVec) {
        typedef u32 u32x2 __attribute__((ext_vector_type(2)));
        typedef u32x2 u32x2_any __attribute__((aligned(1)));
        const u32x2 w = *(const u32x2_any *)(mask_row + tok);  // 8 truth values of one byte
        // byte i's lowest bit to bit 24 + i: no carries, the partial products do not meet
        bits = (((w[0] & 0x01010101u) * 0x01020408u) >> 24 & 0xfu) | (((w[1] & 0x01010101u) * 0x01020408u) >> 20 & 0xf0u);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (i < n && mask_row[tok + i]) bits |= 1u << i;
    }
    return bits;
}

struct RowParams { float rep, inv_rep, pres, freq, inv_temp; };

// z (in: the raw logits; out: the processed ones), slope = d processed / d raw.  `bits`: what the mask allows.
template <bool PEN, bool SLOPE>
__device__ __forceinline__ void process8(float *z, float *slope, u32 bits, const RowParams &p, const u32 *counts8, const void *bias_row,
                                         int bias_kind, i64 tok, int n) {
    if constexpr (SLOPE) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) slope[i] = p.inv_temp;
    }
    if constexpr (PEN) {
        const u32x4 c0 = *(const u32x4 *)counts8, c1 = *(const u32x4 *)(counts8 + kBlk / 2);
        const u32 any = (c0[0] | c0[1] | c0[2]) | (c0[3] | c1[0] | c1[1]) | (c1[2] | c1[3]);
        if (__any(any != 0)) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const u32 c = i < 4 ? c0[i & 3] : c1[i & 3], k = c & ~kSeenInPrompt;
                float f = z[i] > 0.0f ? p.inv_rep : p.rep;
                f = c ? f : 1.0f;
                const float sub = k ? fmaf((float)k, p.freq, p.pres) : 0.0f;
                z[i] = fmaf(z[i], f, -sub);
                if constexpr (SLOPE) slope[i] *= f;
            }
        }
    }
    if (bias_kind != kBiasNone) {
        float b[kVec];
        if (bias_kind == kBiasF32) {
            Raw8<float> r;
            load8((const float *)bias_row + tok, n, r);
            unpack8(r, b);
        } else if (bias_kind == kBiasBf16) {
            Raw8<__bf16> r;
            load8((const __bf16 *)bias_row + tok, n, r);
            unpack8(r, b);
        } else {
            Raw8<_Float16> r;
            load8((const _Float16 *)bias_row + tok, n, r);
            unpack8(r, b);
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) z[i] += b[i];
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        z[i] *= p.inv_temp;
        if (!(bits & (1u << i))) z[i] = neg_inf();
    }
}

__device__ __forceinline__ float wave_max_f(float x) {
    x = fmaxf(x, dpp_mov<0xB1>(x));
    x = fmaxf(x, dpp_mov<0x4E>(x));
    x = fmaxf(x, dpp_mov<0x141>(x));
    x = fmaxf(x, dpp_mov<0x140>(x));
    return fmaxf(fmaxf(read_lane(x, 0), read_lane(x, 16)), fmaxf(read_lane(x, 32), read_lane(x, 48)));
}
__device__ __forceinline__ float wave_sum_f(float x) {
    x += dpp_mov<0xB1>(x);
    x += dpp_mov<0x4E>(x);
    x += dpp_mov<0x141>(x);
    x += dpp_mov<0x140>(x);
    return (read_lane(x, 0) + read_lane(x, 16)) + (read_lane(x, 32) + read_lane(x, 48));
}

// the shift of d = z * log2(e) - shift for a row's (or a wave's) largest value m; *steep: d = (z - m) * log2(e), see the head of the file
__device__ __forceinline__ float softmax_shift(float m, bool *steep) {
    *steep = fabsf(m) >= 0x1p20f && !__builtin_isinf(m);
    return m == neg_inf() || *steep ? 0.0f : m * kLog2e;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T, int MODE, bool PEN, int W>
__global__ __launch_bounds__(W *kWave) void token_kernel(TokenArgs a) {
    constexpr bool kBwd = MODE == kProcessBwd || MODE == kLogProbBwd;
    extern __shared__ __align__(16) u32 lds_counts[];  // PEN: W * kSub words
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const i64 blk = blockIdx.x;
    const i64 slice = blk % a.nslices, rest = blk / a.nslices, chunk = rest % a.nchunks, b = rest / a.nchunks;
    const i64 t0 = chunk * a.chunk, t1 = t0 + a.chunk < a.T ? t0 + a.chunk : a.T;
    const i64 slice_lo = slice * (W * kSub), lo = slice_lo + (i64)wave * kSub;
    u32 *counts = lds_counts + wave * kSub;

    i64 h = 0, prompt = 0;  // history tokens that the counts hold; where the generated ones begin
    if constexpr (PEN) {
        prompt = a.prompt ? load_int(a.prompt, a.prompt_wide, b) : 0;
        u32x4 *c4 = (u32x4 *)lds_counts;
#pragma unroll
        for (int i = 0; i < kSub / 4 / kWave; ++i) c4[threadIdx.x + i * (W * kWave)] = u32x4{0, 0, 0, 0};
        __syncthreads();
        h = a.lengths ? load_int(a.lengths, a.lengths_wide, b * a.T + t0) : a.L;
        h = h < 0 ? 0 : h > a.L ? a.L : h;
        for (i64 j = threadIdx.x; j < h; j += W * kWave)
            count_token(lds_counts, load_int(a.tokens, a.tokens_wide, b * a.tokens_sb + j), slice_lo, W * kSub, j < prompt);
        __syncthreads();
    }
    if (lo >= a.V) return;

    RowParams p;
    p.rep = a.rep_t ? a.rep_t[b] : a.rep;
    p.inv_rep = 1.0f / p.rep;
    p.pres = a.pres_t ? a.pres_t[b] : a.pres;
    p.freq = a.freq_t ? a.freq_t[b] : a.freq;
    p.inv_temp = 1.0f / (a.temp_t ? a.temp_t[b] : a.temp);
    const bool needs_z = MODE != kProcessBwd || (PEN && (a.rep_t || a.rep != 1.0f));

    i64 win_lo = 0;
    i64 win = -1;
    bool have_win = false;

    i64 tok[kRowVecs];
    int nv[kRowVecs];
#pragma unroll
    for (int k = 0; k < kRowVecs; ++k) {
        tok[k] = lo + k * kBlk + lane * kVec;
        const i64 left = a.V - tok[k];
        nv[k] = left > kVec ? kVec : left < 0 ? 0 : (int)left;
    }
    u32 next_bits[kRowVecs];
    const u8 *mask_row = a.mask_kind == TRL_MASK_NONE ? nullptr : (const u8 *)a.mask + b * a.mask_sb + t0 * a.mask_st;
#pragma unroll
    for (int k = 0; k < kRowVecs; ++k) next_bits[k] = mask_bits(a, mask_row, tok[k], nv[k]);

    for (i64 t = t0; t < t1; ++t) {
        const i64 r = b * a.T + t;
        u32 bits[kRowVecs];
#pragma unroll
        for (int k = 0; k < kRowVecs; ++k) bits[k] = next_bits[k];
        if (t + 1 < t1 && a.mask_kind != TRL_MASK_NONE && a.mask_st != 0) {
            const u8 *row = (const u8 *)a.mask + b * a.mask_sb + (t + 1) * a.mask_st;
#pragma unroll
            for (int k = 0; k < kRowVecs; ++k) next_bits[k] = mask_bits(a, row, tok[k], nv[k]);
        }
        // -- the row's scalars
        i64 y = 0;
        float g_lp = 0.0f, ca = 0.0f, cb = 0.0f, shift = 0.0f, top = 0.0f;
        bool zero_row = false, steep = false;
        if constexpr (MODE == kLogProb || MODE == kLogProbBwd) {
            y = load_int(a.action, a.action_wide, r);
            if constexpr (MODE == kLogProb) {
                if (y < 0) continue;  // padding: the joining launch answers for it
            } else {
                const float m = a.stats[2 * r], log2s = a.stats[2 * r + 1];
                zero_row = y < 0 || (m == neg_inf() && log2s == 0.0f);  // a row of NaN has a NaN there
                if (!zero_row) {
                    const float g_h = a.g_entropy ? a.g_entropy[r] : 0.0f, rs = exp2_hw(-log2s);
                    g_lp = a.g_log_prob ? a.g_log_prob[r] : 0.0f;
                    if (y >= a.V) g_lp = __builtin_nanf("");
                    top = m;
                    shift = softmax_shift(m, &steep);
                    ca = rs * (g_lp + g_h * (a.entropy[r] - kLn2 * log2s));
                    cb = rs * g_h * kLn2;
                }
            }
        }
        // -- loads
        const T *z_row = (const T *)a.logits + b * a.logits_sb + t * a.logits_st;
        Raw8<T> zr[kRowVecs], gr[kRowVecs];
#pragma unroll
        for (int k = 0; k < kRowVecs; ++k) {
            zr[k] = Raw8<T>{};
            if (needs_z && bits[k] && !zero_row) load8(z_row + tok[k], nv[k], zr[k]);
            if constexpr (MODE == kProcessBwd) {
                gr[k] = Raw8<T>{};
                if (bits[k]) load8((const T *)a.grad_out + r * a.V + tok[k], nv[k], gr[k]);
            }
        }
        // -- the history grows to this row's
        if constexpr (PEN) {
            i64 want = a.lengths ? load_int(a.lengths, a.lengths_wide, r) : a.L;
            want = want < 0 ? 0 : want > a.L ? a.L : want;
            if (want != h) {
                if (want < h) {  // not a rollout's order: count anew
                    wave_fence();
                    u32x4 *c4 = (u32x4 *)counts;
#pragma unroll
                    for (int i = 0; i < kSub / 4 / kWave; ++i) c4[lane + i * kWave] = u32x4{0, 0, 0, 0};
                    h = 0;
                }
                wave_fence();
                while (h < want) {
                    if (!have_win || h < win_lo || h >= win_lo + kWave) {
                        win_lo = h;
                        have_win = true;
                        const i64 j = h + lane;
                        win = j < a.L ? load_int(a.tokens, a.tokens_wide, b * a.tokens_sb + j) : -1;
                    }
                    const i64 end = want < win_lo + kWave ? want : win_lo + kWave, j = win_lo + lane;
                    if (j >= h && j < end) count_token(counts, win, lo, kSub, j < prompt);
                    h = end;
                }
                wave_fence();
            }
        }
        const void *bias_row = nullptr;
        if (a.bias_kind != kBiasNone) bias_row = (const char *)a.bias + (b * a.bias_sb + t * a.bias_st);

        if constexpr (MODE == kLogProb) {
            float z[kRowVecs][kVec];
            float m = neg_inf();
#pragma unroll
            for (int k = 0; k < kRowVecs; ++k) {
                unpack8(zr[k], z[k]);
                process8<PEN, false>(z[k], nullptr, bits[k], p, counts + k * kBlk + lane * 4, bias_row, a.bias_kind, tok[k], nv[k]);
#pragma unroll
                for (int i = 0; i < kVec; ++i) m = fmaxf(m, z[k][i]);
            }
            m = wave_max_f(m);
            if (y >= lo && y < lo + kSub && y < a.V) {
#pragma unroll
                for (int k = 0; k < kRowVecs; ++k)
#pragma unroll
                    for (int i = 0; i < kVec; ++i)
                        if (tok[k] + i == y) a.z_action[r] = z[k][i];
            }
            bool steep;
            const float shift = softmax_shift(m, &steep);
            if (steep) {
#pragma unroll
                for (int k = 0; k < kRowVecs; ++k)
#pragma unroll
                    for (int i = 0; i < kVec; ++i) z[k][i] -= m;
            }
            float s = 0.0f, u = 0.0f;
#pragma unroll
            for (int k = 0; k < kRowVecs; ++k)
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const float d = fmaf(z[k][i], kLog2e, -shift), e = exp2_hw(d);
                    s += e;
                    u = fmaf(e, fmaxf(d, kFloor), u);
                }
            s = wave_sum_f(s);
            u = wave_sum_f(u);
            if (lane == 0) ((float4 *)a.partials)[r * a.nsubs + lo / kSub] = make_float4(m, s, u, 0.0f);
        } else {
#pragma unroll
            for (int k = 0; k < kRowVecs; ++k) {
                float z[kVec], slope[kVec];
                unpack8(zr[k], z);
                process8<PEN, kBwd>(z, slope, bits[k], p, counts + k * kBlk + lane * 4, MODE == kProcessBwd ? nullptr : bias_row,
                                    MODE == kProcessBwd ? (int)kBiasNone : a.bias_kind, tok[k], bits[k] ? nv[k] : 0);
                if constexpr (MODE == kProcessBwd) {
                    unpack8(gr[k], z);
#pragma unroll
                    for (int i = 0; i < kVec; ++i) z[i] = bits[k] & (1u << i) ? z[i] * slope[i] : 0.0f;
                }
                if constexpr (MODE == kLogProbBwd) {
                    if (steep) {
#pragma unroll
                        for (int i = 0; i < kVec; ++i) z[i] -= top;
                    }
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        const float d = fmaf(z[i], kLog2e, -shift), e = exp2_hw(d);
                        z[i] = -e * fmaf(cb, fmaxf(d, kFloor), ca);
                    }
                    if (y >= lo && y < lo + kSub) {
#pragma unroll
                        for (int i = 0; i < kVec; ++i)
                            if (tok[k] + i == y) z[i] += g_lp;
                    }
#pragma unroll
                    for (int i = 0; i < kVec; ++i) z[i] = (bits[k] & (1u << i)) && !zero_row ? z[i] * slope[i] : 0.0f;
                }
                if (nv[k] > 0) store8((T *)a.out + b * a.out_sb + t * a.out_st + tok[k], nv[k], z);
            }
        }
    }
}

// Joins a row's partials: one wave a row.
__global__ __launch_bounds__(256) void token_join_kernel(TokenArgs a) {
    const int lane = threadIdx.x & (kWave - 1);
    const i64 r = (i64)blockIdx.x * 4 + threadIdx.x / kWave;
    if (r >= a.B * a.T) return;
    const i64 y = load_int(a.action, a.action_wide, r);
    float log_prob = 0.0f, entropy = 0.0f, m = neg_inf(), log2s = 0.0f;
    if (y >= 0) {
        const float4 *part = (const float4 *)a.partials + r * a.nsubs;
        for (i64 i = lane; i < a.nsubs; i += kWave) m = fmaxf(m, part[i].x);
        m = wave_max_f(m);
        bool steep;
        const float shift = softmax_shift(m, &steep);
        float s = 0.0f, u = 0.0f;
        for (i64 i = lane; i < a.nsubs; i += kWave) {
            const float4 q = part[i];
            float d = 0.0f;
            if (q.x != m) {
                bool own;  // whether the wave's values are relative to q.x itself
                const float its = softmax_shift(q.x, &own);
                if (q.x == neg_inf()) d = neg_inf();
                else if (own) d = steep ? (q.x - m) * kLog2e : fmaf(q.x, kLog2e, -shift);
                else d = steep ? fmaf(-m, kLog2e, its) : its - shift;
            }
            const float w = exp2_hw(d);
            s = fmaf(w, q.y, s);
            u = fmaf(w, fmaf(q.y, fmaxf(d, kFloor), q.z), u);
        }
        s = wave_sum_f(s);
        u = wave_sum_f(u);
        if (m == neg_inf() && s == 0.0f) {  // nothing allowed, or nothing possible
            log_prob = neg_inf();
        } else {
            float z = y < a.V ? a.z_action[r] : __builtin_nanf("");
            if (steep) z -= m;
            log2s = log2f(s);
            entropy = kLn2 * (log2s - u / s);
            log_prob = kLn2 * (fmaf(z, kLog2e, -shift) - log2s);
        }
        if (y >= a.V) log_prob = __builtin_nanf("");
    }
    if (lane == 0) {
        a.log_prob[r] = log_prob;
        if (a.entropy) a.entropy[r] = entropy;
        if (a.stats) { a.stats[2 * r] = m; a.stats[2 * r + 1] = log2s; }
    }
}

template <typename T, int MODE, bool PEN, int W>
int launch_w(hipStream_t s, TokenArgs &a) {
    const i64 span = (i64)W * kSub;
    a.nslices = (a.V + span - 1) / span;
    a.nsubs = token_subs(a.V);
    const i64 units = a.nslices * a.B * a.T;
    a.chunk = units / 2048;  // enough blocks for every compute unit, then as long a run of rows as that leaves
    a.chunk = a.chunk < 1 ? 1 : a.chunk > 64 ? 64 : a.chunk;
    if (a.chunk > a.T) a.chunk = a.T;
    a.nchunks = (a.T + a.chunk - 1) / a.chunk;
    const i64 grid = a.nslices * a.nchunks * a.B;
    if (grid > 0x7fffffffLL) return 2;
    hipLaunchKernelGGL((token_kernel<T, MODE, PEN, W>), dim3((unsigned)grid), dim3(W * kWave), PEN ? W * kSub * sizeof(u32) : 0, s, a);
    return 0;
}
template <typename T, int MODE>
int launch_mode(hipStream_t s, TokenArgs &a) {
    return a.tokens ? launch_w<T, MODE, true, 8>(s, a) : launch_w<T, MODE, false, 4>(s, a);
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
    const int rc = launch_dtype<kLogProb>(s, a);
    if (rc) return rc;
    a.nsubs = token_subs(a.V);
    const i64 blocks = (a.B * a.T + 3) / 4;
    if (blocks > 0x7fffffffLL) return 2;
    hipLaunchKernelGGL(token_join_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a);
    return 0;
}
int launch_token_log_prob_bwd(hipStream_t s, TokenArgs a) { return launch_dtype<kLogProbBwd>(s, a); }
