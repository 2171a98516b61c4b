/*
 * TEST INFRASTRUCTURE ONLY -- CPU oracle (see value_oracle_impl.h for the
 * restated algorithms and their reference file:line citations).
 * Parity pin: checked bit-for-bit (GAE, TD(lambda)) / to 2 ulp (V-trace, exp)
 * against the reference imported in the build container and against the golden
 * fixtures under tests/golden/ generated by tools/gen_golden.py.
 *
 * Instantiations: <storage dtype TS>[g<coefficient dtype TG>]
 */
#include <math.h>
#include <stddef.h>

#define TS float
#define TG float
#define TC float
#define SFX f32
#include "value_oracle_impl.h"
#undef TS
#undef TG
#undef TC
#undef SFX

#define TS double
#define TG double
#define TC double
#define SFX f64
#include "value_oracle_impl.h"
#undef TS
#undef TG
#undef TC
#undef SFX

#define TS double
#define TG float
#define TC double
#define SFX f64g32
#include "value_oracle_impl.h"
#undef TS
#undef TG
#undef TC
#undef SFX

#define TS float
#define TG double
#define TC double
#define SFX f32g64
#include "value_oracle_impl.h"
#undef TS
#undef TG
#undef TC
#undef SFX

/* ---------------------------------------------------------------------------
 * Advantage normalisation -- advantages.py:1459-1463 (GAE average_gae),
 * :1828-1832 (VTrace average_adv):  (x - x.mean()) / x.std().clamp_min(eps)
 * with the unbiased (N-1) standard deviation over ALL elements.  Statistics are
 * accumulated in double (two-pass), rounded to the storage dtype, and the scale
 * pass runs in the storage dtype (bit-identical to torch at
 * [65536x32]; torch's own reduction order is internal, so parity is to ~1e-6).
 * stats_out (optional) receives {N, sum, sum of squares} in double.
 * ------------------------------------------------------------------------- */
#define DEF_NORMALIZE(TS, SFX)                                                          \
    void oracle_normalize_##SFX(const TS *x, long n, double eps, TS *out, double *stats_out) \
    {                                                                                   \
        double s = 0.0, ss = 0.0;                                                       \
        for (long k = 0; k < n; ++k) { s += (double)x[k]; ss += (double)x[k] * (double)x[k]; } \
        double mean = n > 0 ? s / (double)n : 0.0;                                      \
        double m2 = 0.0;                                                                \
        for (long k = 0; k < n; ++k) { double d = (double)x[k] - mean; m2 += d * d; }   \
        double var = n > 1 ? m2 / (double)(n - 1) : NAN;                                \
        TS mean_s = (TS)mean;                                                           \
        TS std_s = (TS)sqrt(var);                                                       \
        TS eps_s = (TS)eps;                                                             \
        if (!(std_s >= eps_s) && std_s == std_s) std_s = eps_s; /* clamp_min keeps NaN */ \
        for (long k = 0; k < n; ++k) out[k] = (x[k] - mean_s) / std_s;                  \
        if (stats_out) { stats_out[0] = (double)n; stats_out[1] = s; stats_out[2] = ss; } \
    }
DEF_NORMALIZE(float, f32)
DEF_NORMALIZE(double, f64)

/* ---------------------------------------------------------------------------
 * The benchmark's all-cores CPU baseline: GAE (fp32, scalar coefficients) + normalisation with the env dimension
 * split over OpenMP threads -- per-row sequential loops exactly as oracle_gae_f32 (same operation order, hence the
 * same advantages bit for bit), per-thread fp64 moments, one combine, a parallel scale pass.  The decomposition the
 * GPUs use (shard O, sum {N, sum, sumsq}, scale).  Returns the number of threads used.
 * ------------------------------------------------------------------------- */
#ifdef _OPENMP
#include <omp.h>
#endif
int oracle_gae_normalize_mt_f32(const float *reward, const float *value, const float *next_value,
                                const unsigned char *done, const unsigned char *terminated, double gamma, double lg,
                                long O, long T, double eps, float *advantage, float *value_target, double *stats_out)
{
    double s = 0.0, ss = 0.0;
    int nthreads = 1;
#pragma omp parallel reduction(+ : s, ss)
    {
#ifdef _OPENMP
#pragma omp single
        nthreads = omp_get_num_threads();
#endif
#pragma omp for schedule(static)
        for (long o = 0; o < O; ++o) {
            oracle_gae_f32(reward + o * T, value + o * T, next_value + o * T, done + o * T, terminated + o * T, NULL, NULL,
                           gamma, lg, 1, T, 1, advantage + o * T, value_target + o * T);
            for (long t = 0; t < T; ++t) {
                double a = (double)advantage[o * T + t];
                s += a;
                ss += a * a;
            }
        }
    }
    const double n = (double)O * (double)T;
    const double mean = s / n;
    double var = n > 1 ? (ss - n * mean * mean) / (n - 1.0) : NAN;
    if (var < 0.0) var = 0.0;
    const float mean_s = (float)mean;
    float std_s = (float)sqrt(var);
    const float eps_s = (float)eps;
    if (std_s < eps_s) std_s = eps_s;
#pragma omp parallel for schedule(static)
    for (long k = 0; k < O * T; ++k) advantage[k] = (advantage[k] - mean_s) / std_s;
    if (stats_out) { stats_out[0] = n; stats_out[1] = s; stats_out[2] = ss; }
    return nthreads;
}

int oracle_abi_version(void) { return 2; }
