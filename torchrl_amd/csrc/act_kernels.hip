// Activations kept for the backward pass in 8 bits: trl_act_quantize, trl_act_dequantize, trl_act_weight_grad (include/trl_value.h
// has the format).
#include "act_common.h"
#include "vec8.h"

namespace {

constexpr int kGroups = kActBlock / kVec;  // 4 lanes hold a block

// Thread -> (row, group of 8 features) over N rows of G groups; one 64-bit division a block of threads.
__device__ __forceinline__ bool row_and_group(i64 N, u32 G, i64 &row, u32 &group) {
    const i64 first = (i64)blockIdx.x * blockDim.x;
    const i64 row0 = first / G;
    const u32 off = (u32)(first - row0 * G) + threadIdx.x;
    row = row0 + off / G;
    group = off % G;
    return row < N;
}

// 8 values of a lane to their place `at` (in groups of 8) among the codes.  The four lanes of a block of 32 call together: its largest
// magnitude is two DPP steps; magnitudes are compared as integers, which puts NaN above infinity above every number.
__device__ __forceinline__ void quantize8(const float *v, i64 at, int8_t *codes, u8 *exponents) {
    int top = 0;
#pragma unroll
    for (int i = 0; i < kVec; ++i) top = max(top, __builtin_bit_cast(int, v[i]) & 0x7fffffff);
    top = max(top, dpp_mov<0xB1>(top));
    top = max(top, dpp_mov<0x4E>(top));
    const bool broken = top >= 0x7f800000;
    const int e = max((top >> 23) - 6, 1);
    const float per_step = __builtin_bit_cast(float, (u32)(254 - e) << 23);
    u32 w[2] = {0, 0};
    if (!broken) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int q = (int)rintf(fminf(fmaxf(v[i] * per_step, -127.0f), 127.0f));
            w[i / 4] |= (u32)(q & 0xff) << (8 * (i % 4));
        }
    }
    *(uint2 *)(codes + at * kVec) = make_uint2(w[0], w[1]);
    if ((at & (kGroups - 1)) == 0) exponents[at / kGroups] = (u8)(broken ? 255 : e);
}

// Bound by HBM: 2 bytes in and 1 + 1/32 out an element at 16 bits.  16384 x 8192 bf16: 75-82 us, 5.0-5.4 TB/s (two and four groups of 8 a
// thread with their loads ahead: 75 and 80, dequantizing 79 and 73 against 77; the sum of both is the same within 2 %).
template <typename T>
__global__ __launch_bounds__(256) void act_quantize_kernel(const T *x, i64 stride, i64 N, i64 D, u32 G, int8_t *codes, u8 *exponents) {
    i64 row;
    u32 group;
    if (!row_and_group(N, G, row, group)) return;  // whole blocks of 32 leave together
    const i64 col = (i64)group * kVec, left = D - col;
    Raw8<T> r{};
    const int n = left >= kVec ? kVec : left < 0 ? 0 : (int)left;
    if (n > 0) load8(x + row * stride + col, n, r);
    float v[kVec];
    unpack8(r, v);
    quantize8(v, row * G + group, codes, exponents);
}

// The forward pass of one output (a value head) while its input is quantized: y = x w + b on the way, one read of x.  A wave a row, 512
// features at a time with the next ones on their way; w comes from the caches (two or four rows a wave read it less often, but hide less of
// the latency: 8192 x 4096 bf16 18.7 us and 22.4 / 24.4).  Bound by HBM as the quantization alone: 5.4 TB/s, 19.0 us without the product.
template <typename T, bool KEEP>
__global__ __launch_bounds__(256) void act_head_kernel(const T *__restrict__ x, i64 stride, i64 N, i64 D, u32 G, const T *__restrict__ w, const T *__restrict__ bias,
                                                       int8_t *__restrict__ codes, u8 *__restrict__ exponents, T *__restrict__ y) {
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const i64 row = (i64)blockIdx.x * 4 + wave;
    if (row >= N) return;
    const T *x_row = x + row * stride;
    struct Piece { Raw8<T> x, w; } now, next;
    auto fetch = [&](u32 group) {
        const i64 col = (i64)group * kVec, left = D - col;
        const int n = left >= kVec ? kVec : left < 0 ? 0 : (int)left;
        Piece p{};
        if (n > 0) {
            load8(x_row + col, n, p.x);
            load8(w + col, n, p.w);
        }
        return p;
    };
    float sum = 0.0f;
    auto use = [&](u32 group, const Piece &p) {
        if (group >= G) return;  // whole blocks of 32 leave together
        float v[kVec], vw[kVec];
        unpack8(p.x, v);
        unpack8(p.w, vw);
#pragma unroll
        for (int i = 0; i < kVec; ++i) sum = fmaf(v[i], vw[i], sum);
        if constexpr (KEEP) quantize8(v, row * G + group, codes, exponents);
    };
    now = fetch(lane);
    for (u32 g = 0; g < G; g += 2 * kWave) {
        next = fetch(g + lane + kWave);
        use(g + lane, now);
        now = fetch(g + lane + 2 * kWave);
        use(g + lane + kWave, next);
    }
    sum = wave_sum(sum) + (bias ? (float)bias[0] : 0.0f);
    if (lane == 0) y[row] = (T)sum;
}

__device__ __forceinline__ float step_of(int e) { return e == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, (u32)e << 23); }

// Codes times their step: a product without rounding.  Bound by HBM's writes; 16384 x 8192 bf16: 69 us, 5.9 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void act_dequantize_kernel(const int8_t *codes, const u8 *exponents, i64 N, i64 D, u32 G, T *out) {
    i64 row;
    u32 group;
    if (!row_and_group(N, G, row, group)) return;
    const i64 col = (i64)group * kVec, left = D - col;
    if (left <= 0) return;
    const uint2 w = *(const uint2 *)(codes + (row * G + group) * kVec);
    const float step = step_of(exponents[(row * G + group) / kGroups]);
    float v[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = (float)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i % 4))) * step;
    store8(out + row * D + col, left >= kVec ? kVec : (int)left, v);
}

// ---- dw = dy^T x^ ------------------------------------------------------------------------------------------------------------------
// A (N, O) and a (N, D) matrix, both with the summed dimension outermost, on 32 x 32 x 16 matrix instructions.
//   exact   A code times its step has 7 bits, so x^ is exact in bf16, and in fp16 where it was made from fp16.  dy is used as it is in
//           these types; an fp32 dy is split into three bf16 terms (8 + 8 + 8 bits) that add up to it exactly.  Every product is then
//           exact in the 32-bit accumulators, and the result is off by the sum's own roundings and one to the output type.
//   tiles   The codes go from registers through the conversion into LDS, rows of tokens as in memory; ds_read_tr16 turns 4 x 16 pieces so
//           that a lane gets four consecutive tokens of its own column.  Rows are filled up by 16 elements, so that the four rows of a
//           piece lie in different banks.
//   flow    Two LDS buffers.  While one is multiplied, the next tile goes from registers to the other in the second half of the step, and
//           each register is loaded with the tile after that as soon as it is free: a load has a whole step to arrive, and the
//           conversion runs in the shadow of the matrix instructions.
//   splits  Few output tiles split the tokens; the parts are 32 bits and are added in order by a second launch.
// Bound by the matrix units with a full chip: (8192, 8192)^T (8192, 2048) bf16 takes 255-295 us as the clocks allow, 930-1080 TFLOP/s (the
// library's product of unquantized operands 291), fp32 8192 x 2048 x 2048 299 us (three products; 473).  Partly filled tiles and
// rounds cost the rest: (2048, 3000)^T (2048, 3000) bf16 69 us, 530 TFLOP/s (the library 57-63); 1111 x 515 x 1027 fp32 18 us and 4 to join
// (19 by the library).  One output has a kernel of its own below.
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

template <typename T> constexpr int kTerms = sizeof(T) == 4 ? 3 : 1;

__device__ __forceinline__ u32 high_halves(u32 lo, u32 hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// the bf16 terms of 8 values: term j of elements 2 i and 2 i + 1 in w[j][i]
__device__ __forceinline__ void split8(const float *v, u32x4 *w) {
    float r[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) r[i] = v[i];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        u32 top[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            u32 bits = __builtin_bit_cast(u32, r[i]);
            if (j == 0 && (bits & 0x7fffffffu) > 0x7f800000u) bits |= 0x00400000u;  // a NaN keeps being one without its low half
            top[i] = bits & 0xffff0000u;
            // what is left, exactly; nothing of an infinity or a NaN
            r[i] = (bits & 0x7f800000u) == 0x7f800000u ? 0.0f : r[i] - __builtin_bit_cast(float, top[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) w[j][i] = high_halves(top[2 * i], top[2 * i + 1]);
    }
}

// two exact values as 16 bits each
template <typename T>
__device__ __forceinline__ u32 pack_exact(float lo, float hi) {
    if constexpr (__is_same(T, _Float16)) return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_pkrtz(lo, hi));
    else return high_halves(__builtin_bit_cast(u32, lo), __builtin_bit_cast(u32, hi));
}

// 16 codes times their step, exactly
template <typename T>
__device__ __forceinline__ void convert16(u32x4 codes, int e, u32x4 *w) {
    const float step = step_of(e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const u32 c = codes[i];
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (float)(int8_t)(c >> (8 * k)) * step;
        w[i / 2][2 * (i % 2)] = pack_exact<T>(v[0], v[1]);
        w[i / 2][2 * (i % 2) + 1] = pack_exact<T>(v[2], v[3]);
    }
}

// orders LDS alone: loads from memory stay in flight
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

struct WeightGradArgs {
    const void *dy;
    i64 dy_stride;
    const int8_t *codes;
    const u8 *exponents;
    i64 N, O, D, Dp;
    int tiles_d, tiles;  // output tiles
    i64 part;            // tokens of a split, a multiple of the tile's
    void *dw, *db;       // one split: the outputs
    float *parts;        // more: (splits, O, D) and, behind them, (splits, O)
    int splits;
    const void *w;       // one output alone: the weight and the gradient of the input, or NULL
    void *dx;
};

template <typename T, int BM, int BN, int BK, int WM, int WN>
__global__ __launch_bounds__(WM *WN *kWave, BM == 256 ? 2 : 1) void act_weight_grad_kernel(WeightGradArgs a) {
    constexpr int NT = kTerms<T>, NTHR = WM * WN * kWave;
    constexpr int SA = BM + 16, SB = BN + 16;              // LDS row strides
    constexpr int MI = BM / WM / 32, NI = BN / WN / 32;    // a wave's 32 x 32 pieces
    constexpr int VA = BK * BM / kVec / NTHR, VB = BK * BN / 16 / NTHR;
    constexpr int RA = NTHR / (BM / kVec), RB = NTHR / (BN / 16);  // rows between a thread's vectors
    static_assert(VA * kVec * NTHR == BK * BM && VB * 16 * NTHR == BK * BN && NTHR % (BM / kVec) == 0 && NTHR % (BN / 16) == 0, "whole vectors");
    constexpr int kBuf = BK * (NT * SA + SB);              // elements of a buffer
    extern __shared__ __align__(16) short lds[];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave), wm = wave / WN, wn = wave % WN;

    // consecutive blocks go to the 8 XCDs in turn: give each a run of neighbouring tiles, which share their panels in its L2
    int tile = blockIdx.x % a.tiles;
    const int split = blockIdx.x / a.tiles;
    if (a.tiles % 8 == 0) tile = (tile % 8) * (a.tiles / 8) + tile / 8;
    const i64 o0 = (i64)(tile / a.tiles_d) * BM, d0 = (i64)(tile % a.tiles_d) * BN;
    const i64 n0 = split * a.part, n1 = n0 + a.part < a.N ? n0 + a.part : a.N;
    const bool want_db = a.db && d0 == 0;

    const int a_col = tid % (BM / kVec) * kVec, a_row = tid / (BM / kVec), b_col = tid % (BN / 16) * 16, b_row = tid / (BN / 16);
    const i64 a_left = a.O - (o0 + a_col);
    const int a_n = a_left >= kVec ? kVec : a_left < 0 ? 0 : (int)a_left;
    const bool b_in = d0 + b_col < a.Dp;
    // Whole steps of BK rows below n_whole: a scalar base and a 32-bit offset a vector.  Columns behind the edge end in output elements that
    // are not stored, so any numbers do for them: vectors that lie behind it read the tile's first column, those across it the beginning of
    // the next row -- which the matrix's last row does not have.
    const bool narrow = a.dy_stride >= kVec && a.dy_stride < (1LL << 24) && a.Dp < (1LL << 24);
    const i64 n_last = a.O % kVec && o0 + BM > a.O && n1 == a.N ? n1 - 1 : n1, n_whole = narrow ? n_last : n0;
    const u32 a_off = (u32)(a_row * a.dy_stride + (a_n > 0 ? a_col : 0)) * sizeof(T), a_step = (u32)(RA * a.dy_stride) * sizeof(T);
    const u32 b_off = (u32)(b_row * a.Dp + (b_in ? b_col : 0)), b_step = (u32)(RB * a.Dp);
    Raw8<T> ra[VA];
    u32x4 rb[VB];
    int re[VB];
    auto load_a_whole = [&](i64 n) {
        const char *base = (const char *)a.dy + (n * a.dy_stride + o0) * (i64)sizeof(T);
#pragma unroll
        for (int q = 0; q < VA; ++q) load8((const T *)(base + (a_off + q * a_step)), kVec, ra[q]);
    };
    auto load_b_whole = [&](i64 n) {
        const int8_t *base = a.codes + n * a.Dp + d0;
        const u8 *exps = a.exponents + (n * a.Dp + d0) / kActBlock;
#pragma unroll
        for (int q = 0; q < VB; ++q) {
            rb[q] = *(const u32x4 *)(base + (b_off + q * b_step));
            re[q] = exps[(b_off + q * b_step) / kActBlock];
        }
    };
    auto load_a = [&](i64 n) {
        if (n + BK <= n_whole) load_a_whole(n);
        else {
#pragma unroll
            for (int q = 0; q < VA; ++q) {
                const i64 row = n + a_row + q * RA;
                ra[q] = Raw8<T>{};
                if (row < n1 && a_n > 0) load8((const T *)a.dy + row * a.dy_stride + o0 + a_col, a_n, ra[q]);
            }
        }
    };
    auto load_b = [&](i64 n) {
        if (n + BK <= n_whole) load_b_whole(n);
        else {
#pragma unroll
            for (int q = 0; q < VB; ++q) {
                const i64 row = n + b_row + q * RB;
                rb[q] = u32x4{0, 0, 0, 0};
                re[q] = 127;
                if (row < n1 && b_in) {
                    rb[q] = *(const u32x4 *)(a.codes + row * a.Dp + d0 + b_col);
                    re[q] = a.exponents[(row * a.Dp + d0 + b_col) / kActBlock];
                }
            }
        }
    };
    float col_sum[kVec] = {};
    auto store_a = [&](short *buf, bool sum) {
#pragma unroll
        for (int q = 0; q < VA; ++q) {
            u32x4 w[NT];
            float v[kVec];
            if (NT > 1 || sum) unpack8(ra[q], v);
            if (sum) {
#pragma unroll
                for (int i = 0; i < kVec; ++i) col_sum[i] += v[i];
            }
            if constexpr (NT > 1) split8(v, w);
            else w[0] = ra[q].a;
            short *to = buf + (a_row + q * RA) * (NT * SA) + a_col;
#pragma unroll
            for (int j = 0; j < NT; ++j) *(u32x4 *)(to + j * SA) = w[j];
        }
    };
    auto store_b = [&](short *buf) {
#pragma unroll
        for (int q = 0; q < VB; ++q) {
            u32x4 w[2];
            convert16<T>(rb[q], re[q], w);
            short *to = buf + BK * NT * SA + (b_row + q * RB) * SB + b_col;
            *(u32x4 *)to = w[0];
            *(u32x4 *)(to + 8) = w[1];
        }
    };

    v16f acc[MI][NI] = {};
    // a lane's place in a 16 (tokens) x 32 (columns) piece: see ds_read_tr16 above
    const int fk = (lane / 32) * 8 + (lane % 16) / 4, fc = ((lane / 16) % 2) * 16 + (lane % 4) * 4;
    auto fragment = [&](const short *row0, int stride) {
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(row0 + fk * stride + fc));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(row0 + (fk + 4) * stride + fc));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    if (n0 < n1) {
        load_a(n0);
        load_b(n0);
        store_a(lds, want_db);
        store_b(lds);
        if (n0 + BK < n1) {
            load_a(n0 + BK);
            load_b(n0 + BK);
        }
    }
    __syncthreads();
    int cur = 0;
    i64 n = n0;
    auto multiply = [&](auto fa, auto fb, v16f &c) {
        if constexpr (__is_same(T, _Float16))
            c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, fa), __builtin_bit_cast(v8h, fb), c, 0, 0, 0);
        else
            c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, fa), __builtin_bit_cast(v8bf, fb), c, 0, 0, 0);
    };
    // The long middle, one straight line a step: fragments are fetched one ahead, those of the next step before the step
    // ends.  Two barriers: before the last quarter (the next buffer is written), and before that buffer's successor is written over
    // (every wave is through with the last quarter's reads).
    if constexpr (BK == 64 && NT == 1 && MI % 2 == 0) {
        typedef decltype(fragment(lds, SA)) Frag;
        Frag fa[2], fb[2][NI];
        auto fetch_a = [&](const short *buf, int k, int i) { fa[i % 2] = fragment(buf + k * SA + (wm * MI + i % MI) * 32, SA); };
        auto fetch_b = [&](const short *buf, int k, int to) {
#pragma unroll
            for (int j = 0; j < NI; ++j) fb[to][j] = fragment(buf + BK * SA + k * SB + (wn * NI + j) * 32, SB);
        };
        // 16 tokens at k; the fragments after these come from k2 of buf2
        auto quarter = [&](const short *buf, int k, const short *buf2, int k2, int from) {
            fetch_b(buf2, k2, from ^ 1);
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                if (i + 1 < MI) fetch_a(buf, k, i + 1);
                else fetch_a(buf2, k2, MI);
#pragma unroll
                for (int j = 0; j < NI; ++j) multiply(fa[i % 2], fb[from][j], acc[i][j]);
            }
        };
        auto middle = [&](auto sum) {
            fetch_b(lds, 0, 0);
            fetch_a(lds, 0, 0);
            for (; n + 3 * BK <= n_whole; n += BK, cur ^= 1) {
                const short *buf = lds + cur * kBuf;
                short *next = lds + (cur ^ 1) * kBuf;
                quarter(buf, 0, buf, 16, 0);
                lds_barrier();
                store_a(next, sum.value);
                load_a_whole(n + 2 * BK);
                quarter(buf, 16, buf, 32, 1);
                store_b(next);
                load_b_whole(n + 2 * BK);
                quarter(buf, 32, buf, 48, 0);
                lds_barrier();
                quarter(buf, 48, next, 0, 1);
            }
        };
        if (n + 3 * BK <= n_whole) {
            if (want_db) middle(Bool<true>());
            else middle(Bool<false>());
            __syncthreads();
        }
    }
    for (; n < n1; n += BK, cur ^= 1) {
        const bool more = n + BK < n1, after = n + 2 * BK < n1;
        const short *la = lds + cur * kBuf, *lb = la + BK * NT * SA;
        short *next = lds + (cur ^ 1) * kBuf;
#pragma unroll
        for (int k = 0; k < BK; k += 16) {
            decltype(fragment(lb, SB)) fb[NI];
#pragma unroll
            for (int j = 0; j < NI; ++j) fb[j] = fragment(lb + k * SB + (wn * NI + j) * 32, SB);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const auto fa = fragment(la + k * (NT * SA) + t * SA + (wm * MI + i) * 32, NT * SA);
#pragma unroll
                    for (int j = 0; j < NI; ++j) multiply(fa, fb[j], acc[i][j]);
                }
            if (k == BK - 32 && more) {
                store_a(next, want_db);
                if (after) load_a(n + 2 * BK);
            }
            if (k == BK - 16 && more) {
                store_b(next);
                if (after) load_b(n + 2 * BK);
            }
        }
        __syncthreads();
    }

    // element (row, column) of a piece: row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const i64 d = d0 + (wn * NI + j) * 32 + lane % 32;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const i64 o = o0 + (wm * MI + i) * 32 + 8 * (r / 4) + 4 * (lane / 32) + r % 4;
                if (o < a.O && d < a.D) {
                    if (a.splits == 1) ((T *)a.dw)[o * a.D + d] = (T)acc[i][j][r];
                    else a.parts[((i64)split * a.O + o) * a.D + d] = acc[i][j][r];
                }
            }
        }
    if (want_db) {  // the block's threads of a column group, added in order (the loop's last barrier has freed the buffers)
        float *sums = (float *)lds;
#pragma unroll
        for (int i = 0; i < kVec; ++i) sums[a_row * BM + a_col + i] = col_sum[i];
        __syncthreads();
        for (int c = tid; c < BM; c += NTHR) {
            float s = 0.0f;
            for (int r = 0; r < RA; ++r) s += sums[r * BM + c];
            if (o0 + c < a.O) {
                if (a.splits == 1) ((T *)a.db)[o0 + c] = (T)s;
                else a.parts[(i64)a.splits * a.O * a.D + (i64)split * a.O + o0 + c] = s;
            }
        }
    }
}

// Adds the parts of a split sum in a fixed order; bound by a launch's latency.  Few parts: a thread a column (3 parts of 515 x 1027: 4.1 us,
// 7.4 with 8 threads a column).  Many: 8 threads a column, a share of the parts each (256 parts of 256 columns: 5 us and 13).
constexpr int kFewParts = 16;
template <typename T, int GROUPS>
__global__ __launch_bounds__(256) void act_join_kernel(const float *parts, int splits, i64 n_w, i64 n_b, T *dw, T *db) {
    constexpr int kCols = 256 / GROUPS;
    const int col = threadIdx.x % kCols, group = threadIdx.x / kCols;
    const i64 i = (i64)blockIdx.x * kCols + col;
    const bool in = i < n_w + n_b, w = i < n_w;
    const i64 n = w ? n_w : n_b, at = w ? i : i - n_w;
    const float *p = parts + (w ? 0 : splits * n_w) + at;
    float s = 0.0f;
    if (in) {
#pragma unroll 8
        for (int k = group; k < splits; k += GROUPS) s += p[k * n];
    }
    if constexpr (GROUPS > 1) {
        __shared__ float sums[GROUPS][kCols];
        sums[group][col] = s;
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int k = 1; k < GROUPS; ++k) s += sums[k][col];
    }
    if (in) (w ? dw : db)[at] = (T)s;
}

// The backward pass of one output (a value head): dw is a column sum of x^ weighted by dy, one read of the codes, and dx = dy w is written
// beside it.  A wave takes 512 columns, 8 a lane, and every 8th row of its split, kHeadRows at a time; dy of 64 rows lies in its lanes.
// Products are exact in the fma.  Bound by HBM: 8192 x 4096 bf16 25 us with the join of 32 parts (4.0 TB/s), 15 without dx; 65536 x 1024
// 36 us (5.6 TB/s).  8 and 16 rows at a time: 25.5 / 23.7 us, but 65536 x 1024 37.5 / 38.8 and 8192 x 16384 89 / 102 against 85.
constexpr int kHeadRows = 4, kHeadWaves = 8, kHeadCols = kVec * kWave;
template <typename T>
__global__ __launch_bounds__(kHeadWaves * kWave) void act_head_grad_kernel(WeightGradArgs a) {
    __shared__ float sums[kHeadWaves][kHeadCols + 1];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const i64 d0 = (i64)(blockIdx.x % a.tiles) * kHeadCols + lane * kVec;
    const int split = blockIdx.x / a.tiles;
    const i64 n0 = split * a.part, n1 = n0 + a.part < a.N ? n0 + a.part : a.N;
    const bool in = d0 < a.Dp;
    const i64 left = a.D - d0;
    const int n_dx = !a.dx ? 0 : left >= kVec ? kVec : left < 0 ? 0 : (int)left;
    Raw8<T> rw{};
    if (n_dx > 0) load8((const T *)a.w + d0, n_dx, rw);
    float w[kVec], s[kVec] = {}, s_dy = 0.0f;
    unpack8(rw, w);
    for (i64 n = n0 + wave; n < n1; n += kHeadWaves * kWave) {
        const i64 mine = n + lane * kHeadWaves;
        const float dy = mine < n1 ? (float)((const T *)a.dy)[mine * a.dy_stride] : 0.0f;
        s_dy += dy;
        const i64 ahead = (n1 - n + kHeadWaves - 1) / kHeadWaves;
        const int rows = ahead < kWave ? (int)ahead : kWave;
        for (int k0 = 0; k0 < rows; k0 += kHeadRows) {
            uint2 c[kHeadRows];
            int e[kHeadRows];
#pragma unroll
            for (int k = 0; k < kHeadRows; ++k) {
                c[k] = make_uint2(0, 0);
                e[k] = 127;
                const i64 at = (n + (i64)(k0 + k) * kHeadWaves) * a.Dp + d0;
                if (k0 + k < rows && in) {
                    c[k] = *(const uint2 *)(a.codes + at);
                    e[k] = a.exponents[at / kActBlock];
                }
            }
#pragma unroll
            for (int k = 0; k < kHeadRows; ++k) {
                const float g = k0 + k < rows ? read_lane(dy, k0 + k) : 0.0f, step = step_of(e[k]);
#pragma unroll
                for (int i = 0; i < kVec; ++i) s[i] = fmaf(g, (float)(int8_t)((i < 4 ? c[k].x : c[k].y) >> (8 * (i % 4))) * step, s[i]);
                if (n_dx > 0 && k0 + k < rows) {
                    float dx[kVec];
#pragma unroll
                    for (int i = 0; i < kVec; ++i) dx[i] = g * w[i];
                    store8((T *)a.dx + (n + (i64)(k0 + k) * kHeadWaves) * a.D + d0, n_dx, dx);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) sums[wave][lane * kVec + i] = s[i];
    s_dy = wave_sum(s_dy);
    if (lane == 0) sums[wave][kHeadCols] = s_dy;
    __syncthreads();
    const i64 d = (i64)(blockIdx.x % a.tiles) * kHeadCols + threadIdx.x;
    auto total = [&](int c) {
        float t = 0.0f;
#pragma unroll
        for (int w = 0; w < kHeadWaves; ++w) t += sums[w][c];
        return t;
    };
    if (d < a.D) {
        if (a.splits == 1) ((T *)a.dw)[d] = (T)total(threadIdx.x);
        else a.parts[(i64)split * a.D + d] = total(threadIdx.x);
    }
    if (a.db && blockIdx.x % a.tiles == 0 && threadIdx.x == 0) {
        if (a.splits == 1) ((T *)a.db)[0] = (T)total(kHeadCols);
        else a.parts[(i64)a.splits * a.D + split] = total(kHeadCols);
    }
}

// Column sums of dy alone: 32 groups of 8 columns a block, 8 rows at a time.
template <typename T>
__global__ __launch_bounds__(256) void act_column_sum_kernel(WeightGradArgs a) {
    __shared__ float sums[8][256];
    const i64 o0 = (i64)(blockIdx.x % a.tiles) * 256;
    const int split = blockIdx.x / a.tiles, col = threadIdx.x % 32 * kVec, row = threadIdx.x / 32;
    const i64 left = a.O - (o0 + col), n0 = split * a.part, n1 = n0 + a.part < a.N ? n0 + a.part : a.N;
    const int n_col = left >= kVec ? kVec : left < 0 ? 0 : (int)left;
    float s[kVec] = {};
    if (n_col > 0) {
        for (i64 n = n0 + row; n < n1; n += 8) {
            Raw8<T> r{};
            load8((const T *)a.dy + n * a.dy_stride + o0 + col, n_col, r);
            float v[kVec];
            unpack8(r, v);
#pragma unroll
            for (int i = 0; i < kVec; ++i) s[i] += v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) sums[row][col + i] = s[i];
    __syncthreads();
    const i64 o = o0 + threadIdx.x;
    if (o >= a.O) return;
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += sums[k][threadIdx.x];
    if (a.splits == 1) ((T *)a.db)[o] = (T)t;
    else a.parts[(i64)split * a.O + o] = t;
}

// Tile and splits: the cheapest of a few by a count of clocks.  A block costs `clocks` a token (measured with the chip full, `slots`
// blocks at a time; the head and tail of a block as two steps more), the parts of a split sum are written and read at 1900 bytes a clock,
// and joining them is a launch of its own.  By the count and measured, us at 2.4 GHz without the join: 8192 x 2048 x 8192 bf16 267 and 260-282,
// 8192 x 2048 x 2048 fp32 277 and 257-275, 65536 x 257 x 13 bf16 25 and 22, fp32 38 and 29.
struct WeightGradPlan { int bm, bn, bk; i64 tiles_d, tiles, part; int splits; };
WeightGradPlan weight_grad_plan(int dtype, i64 N, i64 O, i64 D) {
    WeightGradPlan p{};
    if (D == 0) {  // column sums alone
        p.tiles = (O + 255) / 256;
        const i64 want = (512 + p.tiles - 1) / p.tiles, most = (N + 127) / 128 > 0 ? (N + 127) / 128 : 1;
        p.part = N / (want < most ? want : most) + 1;
        p.splits = (int)(N ? (N + p.part - 1) / p.part : 1);
        return p;
    }
    if (O == 1) {  // a value head: enough blocks for the chip, 64 rows or more a split
        p.tiles = (D + kHeadCols - 1) / kHeadCols;
        const i64 want = (256 + p.tiles - 1) / p.tiles, most = (N + 63) / 64 > 0 ? (N + 63) / 64 : 1, s = want < most ? want : most;
        p.part = (N + s - 1) / s + (N == 0);
        p.splits = (int)(N ? (N + p.part - 1) / p.part : 1);
        return p;
    }
    struct Tile { int bm, bn, bk, slots; double clocks; };
    static const Tile low[] = {{256, 256, 64, 256, 77.0}, {128, 128, 64, 512, 52.0}, {32, 128, 64, 768, 55.0}};
    static const Tile f32[] = {{128, 128, 32, 512, 160.0}, {32, 128, 64, 512, 80.0}};
    const Tile *from = dtype == TRL_F32 ? f32 : low, *to = dtype == TRL_F32 ? f32 + 2 : low + 3;
    double best = 0.0;
    for (const Tile *t = from; t < to; ++t) {
        const i64 tiles_d = (D + t->bn - 1) / t->bn, tiles = tiles_d * ((O + t->bm - 1) / t->bm);
        for (i64 s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
            i64 part = ((N + s - 1) / s + t->bk - 1) / t->bk * t->bk;
            if (part == 0) part = t->bk;
            const i64 splits = N ? (N + part - 1) / part : 1;
            if (s > 1 && (part < 2 * t->bk || splits < 2)) break;
            const i64 rounds = (tiles * splits + t->slots - 1) / t->slots;
            const double cost = (double)rounds * (double)(part + 2 * t->bk) * t->clocks + (splits > 1 ? (double)splits * (double)(O * D) * 8.0 / 1900.0 + 9000.0 : 0.0);
            if (p.splits == 0 || cost < best) {
                best = cost;
                p = {t->bm, t->bn, t->bk, tiles_d, tiles, part, (int)splits};
            }
        }
    }
    return p;
}

template <typename T, int BM, int BN, int BK, int WM, int WN>
void launch_weight_grad(hipStream_t s, const WeightGradArgs &a) {
    constexpr size_t bytes = 2 * sizeof(short) * BK * (kTerms<T> * (BM + 16) + BN + 16);
    static_assert(bytes <= 160 * 1024 && bytes >= sizeof(float) * kVec * WM * WN * kWave, "LDS: two buffers, and the column sums after them");
    hipLaunchKernelGGL((act_weight_grad_kernel<T, BM, BN, BK, WM, WN>), dim3((unsigned)(a.tiles * a.splits)), dim3(WM * WN * kWave), bytes, s, a);
}
template <typename T>
void launch_weight_grad_t(hipStream_t s, const WeightGradArgs &a, const WeightGradPlan &p) {
    if (a.D == 0) hipLaunchKernelGGL(act_column_sum_kernel<T>, dim3((unsigned)(a.tiles * a.splits)), dim3(256), 0, s, a);
    else if (a.O == 1) hipLaunchKernelGGL(act_head_grad_kernel<T>, dim3((unsigned)(a.tiles * a.splits)), dim3(kHeadWaves * kWave), 0, s, a);
    else if (p.bm == 32) launch_weight_grad<T, 32, 128, 64, 1, 4>(s, a);
    else if constexpr (sizeof(T) == 4) launch_weight_grad<T, 128, 128, 32, 2, 2>(s, a);
    else {
        if (p.bm == 256) launch_weight_grad<T, 256, 256, 64, 2, 4>(s, a);
        else launch_weight_grad<T, 128, 128, 64, 2, 2>(s, a);
    }
    if (a.splits > 1) {
        const i64 n_w = a.O * a.D, n_b = a.db ? a.O : 0;
        auto join = [&](auto kernel, int cols) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((n_w + n_b + cols - 1) / cols)), dim3(256), 0, s, a.parts, a.splits, n_w, n_b, (T *)a.dw, (T *)a.db);
        };
        if (a.splits > kFewParts) join(act_join_kernel<T, 8>, 32);
        else join(act_join_kernel<T, 1>, 256);
    }
}

}  // namespace

// Calls launch(first row, rows) on runs of rows that one launch can take, `each` being the threads of one.
template <typename F>
static void in_launches(i64 N, i64 each, F launch) {
    const i64 most = kMostThreads / each;
    for (i64 r = 0; r < N; r += most) launch(r, N - r < most ? N - r : most);
}

void launch_act_quantize(hipStream_t s, int dtype, const void *x, i64 stride, i64 N, i64 D, int8_t *codes, u8 *exponents) {
    const u32 G = (u32)((D + kActBlock - 1) / kActBlock * kGroups);
    auto launch = [&](auto t) {
        typedef decltype(t) T;
        in_launches(N, G, [&](i64 r, i64 n) {
            hipLaunchKernelGGL(act_quantize_kernel<T>, dim3((unsigned)((n * G + 255) / 256)), dim3(256), 0, s, (const T *)x + r * stride, stride, n, D, G,
                               codes + r * G * kVec, exponents + r * G / kGroups);
        });
    };
    if (dtype == TRL_F32) launch(0.0f);
    else if (dtype == TRL_BF16) launch((__bf16)0.0f);
    else launch((_Float16)0.0f);
}

void launch_act_dequantize(hipStream_t s, int dtype, const int8_t *codes, const u8 *exponents, i64 N, i64 D, void *out) {
    const u32 G = (u32)((D + kActBlock - 1) / kActBlock * kGroups);
    auto launch = [&](auto t) {
        typedef decltype(t) T;
        in_launches(N, G, [&](i64 r, i64 n) {
            hipLaunchKernelGGL(act_dequantize_kernel<T>, dim3((unsigned)((n * G + 255) / 256)), dim3(256), 0, s, codes + r * G * kVec,
                               exponents + r * G / kGroups, n, D, G, (T *)out + r * D);
        });
    };
    if (dtype == TRL_F32) launch(0.0f);
    else if (dtype == TRL_BF16) launch((__bf16)0.0f);
    else launch((_Float16)0.0f);
}

size_t act_weight_grad_workspace(int dtype, i64 N, i64 O, i64 D) {
    const WeightGradPlan p = weight_grad_plan(dtype, N, O, D);
    return p.splits > 1 ? (size_t)p.splits * (size_t)O * (size_t)(D + 1) * sizeof(float) : 0;  // parts of dw, then of db
}

void launch_act_head(hipStream_t s, int dtype, const void *x, i64 stride, i64 N, i64 D, const void *w, const void *bias, int8_t *codes, u8 *exponents, void *y) {
    const u32 G = (u32)((D + kActBlock - 1) / kActBlock * kGroups);
    auto launch = [&](auto t) {
        typedef decltype(t) T;
        const auto kernel = codes ? act_head_kernel<T, true> : act_head_kernel<T, false>;
        in_launches(N, kWave, [&](i64 r, i64 n) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, s, (const T *)x + r * stride, stride, n, D, G, (const T *)w,
                               (const T *)bias, codes ? codes + r * G * kVec : nullptr, codes ? exponents + r * G / kGroups : nullptr, (T *)y + r);
        });
    };
    if (dtype == TRL_F32) launch(0.0f);
    else if (dtype == TRL_BF16) launch((__bf16)0.0f);
    else launch((_Float16)0.0f);
}

int launch_act_weight_grad(hipStream_t s, int dtype, const void *dy, i64 dy_stride, const int8_t *codes, const u8 *exponents, i64 N, i64 O,
                           i64 D, void *dw, void *db, void *workspace, const void *w, void *dx) {
    const WeightGradPlan p = weight_grad_plan(dtype, N, O, D);
    // 512 threads a block at most; parts of a split sum are joined by up to 8 a column
    if (p.tiles * p.splits > kMostThreads / 512 || (p.splits > 1 && O * (D + 1) > kMostThreads / (p.splits > kFewParts ? 8 : 1))) return 2;
    const WeightGradArgs a{dy, dy_stride, codes, exponents, N, O, D, (D + kActBlock - 1) / kActBlock * kActBlock, (int)p.tiles_d, (int)p.tiles, p.part, dw, db,
                           (float *)workspace, p.splits, w, dx};
    if (dtype == TRL_F32) launch_weight_grad_t<float>(s, a, p);
    else if (dtype == TRL_BF16) launch_weight_grad_t<__bf16>(s, a, p);
    else launch_weight_grad_t<_Float16>(s, a, p);
    return 0;
}
