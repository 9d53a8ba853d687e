// rope_freq.h -- the inverse frequencies of rotary positions (buildRopeInvFreq
// model.go:1728-1756, YaRN :1758-1799) in 64 bits.  Host arithmetic only.
#pragma once

#include <math.h>

#include "../../include/gllm_hip.h"

namespace gllm {

// inv[0 .. rot_dim / 2) and the amplitude of a checked configuration.
//   plain   inv_i = theta^(-2 i / rot_dim)
//   linear  inv_i / factor
//   llama3  inv_i where a wave fits orig_ctx more than high_freq_factor times,
//           inv_i / factor where less than low_freq_factor times, and a
//           mixture, linear in the number of turns, between
//   yarn    inv_i below the dimension that turns beta_fast times in orig_ctx,
//           inv_i / factor above the one that turns beta_slow times, and a
//           mixture, linear in i, between; amplitude
//           attn_factor * (0.1 ln(factor) + 1), and attn_factor for the others
// each divided by freq_factors[i] where given.
inline void rope_frequencies(const gllm_hip_rope_config& c, double* inv, double* amp) {
    const double two_pi = 6.283185307179586476925;
    const int half = c.rot_dim / 2;
    double lo = 0, hi = 0;
    *amp = c.attn_factor;
    if (c.scaling == GLLM_ROPE_YARN) {
        const auto dim = [&](double turns) {
            return c.rot_dim * log(c.orig_ctx / (turns * two_pi)) / (2 * log(c.theta));
        };
        lo = fmax(floor(dim(c.beta_fast)), 0.0);
        hi = fmin(ceil(dim(c.beta_slow)), c.rot_dim - 1.0);
        *amp *= 0.1 * log(c.factor) + 1.0;
    }
    for (int i = 0; i < half; i++) {
        double f = pow(c.theta, -2.0 * i / c.rot_dim);
        if (c.scaling == GLLM_ROPE_LINEAR) {
            f /= c.factor;
        } else if (c.scaling == GLLM_ROPE_LLAMA3) {
            const double turns = c.orig_ctx * f / two_pi;
            const double t = fmin(fmax((turns - c.low_freq_factor) / (c.high_freq_factor - c.low_freq_factor), 0.0), 1.0);
            f *= (1.0 - t) / c.factor + t;
        } else if (c.scaling == GLLM_ROPE_YARN) {
            const double t = fmin(fmax((i - lo) / fmax(hi - lo, 1e-3), 0.0), 1.0);
            f *= t / c.factor + (1.0 - t);
        }
        inv[i] = c.freq_factors ? f / (double)c.freq_factors[i] : f;
    }
}

// Why a configuration is not usable, or null.
inline const char* rope_config_error(const gllm_hip_rope_config& c) {
    const auto pos = [](double v) { return isfinite(v) && v > 0; };
    if (c.head_dim < 2 || c.head_dim > 1024) return "head_dim must be 2..1024";
    if (c.rot_dim < 2 || c.rot_dim % 2 || c.rot_dim > c.head_dim) return "rot_dim must be even, 2..head_dim";
    if (c.layout != GLLM_ROPE_INTERLEAVED && c.layout != GLLM_ROPE_HALF) return "unknown layout";
    if (!(isfinite(c.theta) && c.theta > 1)) return "theta must be finite and > 1";
    if (!pos(c.attn_factor)) return "attn_factor must be finite and > 0";
    if (c.scaling < GLLM_ROPE_PLAIN || c.scaling > GLLM_ROPE_LLAMA3) return "unknown scaling";
    if (c.scaling != GLLM_ROPE_PLAIN && !(pos(c.factor) && c.factor >= 1)) return "factor must be finite and >= 1";
    if (c.scaling == GLLM_ROPE_YARN || c.scaling == GLLM_ROPE_LLAMA3) {
        if (c.orig_ctx < 1) return "orig_ctx must be >= 1";
        if (c.scaling == GLLM_ROPE_YARN && !(pos(c.beta_slow) && pos(c.beta_fast) && c.beta_fast >= c.beta_slow))
            return "beta_fast >= beta_slow > 0 is needed";
        if (c.scaling == GLLM_ROPE_LLAMA3 &&
            !(pos(c.low_freq_factor) && pos(c.high_freq_factor) && c.high_freq_factor > c.low_freq_factor))
            return "high_freq_factor > low_freq_factor > 0 is needed";
    }
    if (c.freq_factors)
        for (int i = 0; i < c.rot_dim / 2; i++)
            if (!(pos(c.freq_factors[i]) && c.freq_factors[i] >= 1e-3f)) return "freq_factors must be finite and >= 0.001";
    return nullptr;
}

}  // namespace gllm
