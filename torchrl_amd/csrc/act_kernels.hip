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

// Bound by HBM: 2 bytes in and 1 + 1/32 out an element at 16 bits.  Four lanes hold a block of 32, so its largest magnitude is two
// DPP steps; magnitudes are compared as integers, which puts NaN above infinity above every number.
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
    *(uint2 *)(codes + (row * G + group) * kVec) = make_uint2(w[0], w[1]);
    if ((group & (kGroups - 1)) == 0) exponents[(row * G + group) / kGroups] = (u8)(broken ? 255 : e);
}

__device__ __forceinline__ float step_of(int e) { return e == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, (u32)e << 23); }

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

// dw = dy^T x^, one 64 x 64 tile a block, 4 x 4 values a thread.
template <typename T>
__global__ __launch_bounds__(256) void act_weight_grad_kernel(const T *dy, i64 dy_stride, const int8_t *codes, const u8 *exponents, i64 N, i64 O,
                                                              i64 D, i64 Dp, i64 tiles_d, T *dw, T *db) {
    constexpr int BM = 64, BN = 64, BK = 16;
    __shared__ float sa[BK][BM], sb[BK][BN];
    const i64 o0 = (blockIdx.x / tiles_d) * BM, d0 = (blockIdx.x % tiles_d) * BN;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {}, bias[4] = {};
    for (i64 n0 = 0; n0 < N; n0 += BK) {
        for (int i = threadIdx.x; i < BK * BM; i += 256) {
            const i64 n = n0 + i / BM, o = o0 + i % BM;
            sa[i / BM][i % BM] = n < N && o < O ? (float)dy[n * dy_stride + o] : 0.0f;
        }
        for (int i = threadIdx.x; i < BK * BN; i += 256) {
            const i64 n = n0 + i / BN, d = d0 + i % BN;
            sb[i / BN][i % BN] = n < N && d < Dp ? (float)codes[n * Dp + d] * step_of(exponents[(n * Dp + d) / kActBlock]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < BK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bias[i] += sa[k][ty * 4 + i];
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
            }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const i64 o = o0 + ty * 4 + i;
        if (o >= O) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (d0 + tx * 4 + j < D) dw[o * D + d0 + tx * 4 + j] = (T)acc[i][j];
        if (db && d0 == 0 && tx == 0) db[o] = (T)bias[i];
    }
}

}  // namespace

void launch_act_quantize(hipStream_t s, int dtype, const void *x, i64 stride, i64 N, i64 D, int8_t *codes, u8 *exponents) {
    const u32 G = (u32)((D + kActBlock - 1) / kActBlock * kGroups);
    const dim3 grid((unsigned)((N * G + 255) / 256));
    if (dtype == TRL_F32) hipLaunchKernelGGL(act_quantize_kernel<float>, grid, dim3(256), 0, s, (const float *)x, stride, N, D, G, codes, exponents);
    else if (dtype == TRL_BF16) hipLaunchKernelGGL(act_quantize_kernel<__bf16>, grid, dim3(256), 0, s, (const __bf16 *)x, stride, N, D, G, codes, exponents);
    else hipLaunchKernelGGL(act_quantize_kernel<_Float16>, grid, dim3(256), 0, s, (const _Float16 *)x, stride, N, D, G, codes, exponents);
}

void launch_act_dequantize(hipStream_t s, int dtype, const int8_t *codes, const u8 *exponents, i64 N, i64 D, void *out) {
    const u32 G = (u32)((D + kActBlock - 1) / kActBlock * kGroups);
    const dim3 grid((unsigned)((N * G + 255) / 256));
    if (dtype == TRL_F32) hipLaunchKernelGGL(act_dequantize_kernel<float>, grid, dim3(256), 0, s, codes, exponents, N, D, G, (float *)out);
    else if (dtype == TRL_BF16) hipLaunchKernelGGL(act_dequantize_kernel<__bf16>, grid, dim3(256), 0, s, codes, exponents, N, D, G, (__bf16 *)out);
    else hipLaunchKernelGGL(act_dequantize_kernel<_Float16>, grid, dim3(256), 0, s, codes, exponents, N, D, G, (_Float16 *)out);
}

size_t act_weight_grad_workspace(int dtype, i64 N, i64 O, i64 D) { return 0; }

int launch_act_weight_grad(hipStream_t s, int dtype, const void *dy, i64 dy_stride, const int8_t *codes, const u8 *exponents, i64 N, i64 O,
                           i64 D, void *dw, void *db, void *workspace) {
    const i64 Dp = (D + kActBlock - 1) / kActBlock * kActBlock, tiles_d = (D + 63) / 64, tiles = tiles_d * ((O + 63) / 64);
    if (tiles > 0x7fffffffLL) return 2;
    const dim3 grid((unsigned)tiles);
    if (dtype == TRL_F32)
        hipLaunchKernelGGL(act_weight_grad_kernel<float>, grid, dim3(256), 0, s, (const float *)dy, dy_stride, codes, exponents, N, O, D, Dp, tiles_d, (float *)dw, (float *)db);
    else if (dtype == TRL_BF16)
        hipLaunchKernelGGL(act_weight_grad_kernel<__bf16>, grid, dim3(256), 0, s, (const __bf16 *)dy, dy_stride, codes, exponents, N, O, D, Dp, tiles_d, (__bf16 *)dw, (__bf16 *)db);
    else
        hipLaunchKernelGGL(act_weight_grad_kernel<_Float16>, grid, dim3(256), 0, s, (const _Float16 *)dy, dy_stride, codes, exponents, N, O, D, Dp, tiles_d, (_Float16 *)dw, (_Float16 *)db);
    return 0;
}
