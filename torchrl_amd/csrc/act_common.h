// Launchers of the 8-bit activation kernels (act_kernels.hip), called from capi.hip.
#pragma once
#include "../../include/trl_value.h"
#include "common.h"

constexpr int kActBlock = 32;  // features that share a step

void launch_act_quantize(hipStream_t s, int dtype, const void *x, i64 stride, i64 N, i64 D, int8_t *codes, u8 *exponents);
void launch_act_dequantize(hipStream_t s, int dtype, const int8_t *codes, const u8 *exponents, i64 N, i64 D, void *out);
size_t act_weight_grad_workspace(int dtype, i64 N, i64 O, i64 D);
// 0, or 2 where the grid would pass its limit
int launch_act_weight_grad(hipStream_t s, int dtype, const void *dy, i64 dy_stride, const int8_t *codes, const u8 *exponents, i64 N, i64 O,
                           i64 D, void *dw, void *db, void *workspace, const void *w = nullptr, void *dx = nullptr);
void launch_act_head(hipStream_t s, int dtype, const void *x, i64 stride, i64 N, i64 D, const void *w, const void *bias, int8_t *codes, u8 *exponents, void *y);
