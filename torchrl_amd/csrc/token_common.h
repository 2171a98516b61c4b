// Parameter block and launchers of the token-policy kernels (token_kernels.hip), called from capi.hip.
#pragma once
#include "../../include/trl_value.h"
#include "common.h"

enum { kBiasNone = 0, kBiasF32 = 1 + TRL_F32, kBiasBf16 = 1 + TRL_BF16, kBiasF16 = 1 + TRL_F16 };

// Rows are (b, t) of B sequences with T rows each, row index r = b * T + t.
struct TokenArgs : trl_token_args {
    float *partials, *z_action;              // workspace of the forward call: (B * T, nsubs, 4), (B * T,)
    int64_t nslices, nchunks, chunk, nsubs;  // set by the launcher
};

i64 token_subs(i64 V);  // sub-slices of a vocabulary: the partials of a row
// 0, or 2 where the grid would pass its limit
int launch_process_logits(hipStream_t s, TokenArgs a);
int launch_process_logits_bwd(hipStream_t s, TokenArgs a);
int launch_token_log_prob(hipStream_t s, TokenArgs a);
int launch_token_log_prob_bwd(hipStream_t s, TokenArgs a);
