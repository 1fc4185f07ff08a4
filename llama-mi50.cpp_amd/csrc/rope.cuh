// rope.cuh — the angles of ROPE / ROPE_BACK, shared by every kernel that rotates.
#pragma once

#include "common.h"
#include <cmath>

namespace mx {

struct RopeP {
    int n_dims, mode;
    float freq_scale, ext_factor, attn_factor, theta_scale;
    float corr0, corr1;
    // several axes (mode & GGML_ROPE_TYPE_MROPE), and the sign of the sine (-1: ROPE_BACK)
    int sect[4];
    float sin_sign;
    double log2_base;
};

static inline bool rope_has_axes(int mode) { return (mode & GGML_ROPE_TYPE_MROPE) != 0; }
// channel pairs that turn; VISION's n_dims is half the head, and all of it turns
static inline int rope_pairs(int mode, int n_dims) { return mode == GGML_ROPE_TYPE_VISION ? n_dims : n_dims / 2; }
constexpr int MX_ROPE_MAXP = 512;     // pairs of a token's cos / sin table in LDS

static inline float yarn_corr_dim(int n_dims, int n_ctx_orig, float n_rot, float base) {
    return n_dims * logf(n_ctx_orig / (n_rot * 2 * (float) M_PI)) / (2 * logf(base));
}

// op_params of a ROPE / ROPE_BACK node (ggml.c ggml_rope_impl)
static inline RopeP rope_params(const ggml_tensor * dst) {
    RopeP p;
    p.n_dims = mx_op_param<int32_t>(dst, 1);
    p.mode = mx_op_param<int32_t>(dst, 2);
    const int n_ctx_orig = mx_op_param<int32_t>(dst, 4);
    const float freq_base = mx_op_param<float>(dst, 5);
    p.freq_scale = mx_op_param<float>(dst, 6);
    p.ext_factor = mx_op_param<float>(dst, 7);
    p.attn_factor = mx_op_param<float>(dst, 8);
    const float beta_fast = mx_op_param<float>(dst, 9), beta_slow = mx_op_param<float>(dst, 10);
    p.theta_scale = powf(freq_base, -2.0f / p.n_dims);
    const float start = floorf(yarn_corr_dim(p.n_dims, n_ctx_orig, beta_fast, freq_base));
    const float end = ceilf(yarn_corr_dim(p.n_dims, n_ctx_orig, beta_slow, freq_base));
    p.corr0 = fmaxf(0.0f, start);
    p.corr1 = fminf((float) (p.n_dims - 1), end);
    for (int i = 0; i < 4; ++i) p.sect[i] = mx_op_param<int32_t>(dst, 11 + i);
    p.log2_base = log2((double) freq_base);
    p.sin_sign = dst->op == GGML_OP_ROPE_BACK ? -1.0f : 1.0f;
    return p;
}

// ROPE of one axis by a workgroup a token rather than a row (op_rope, ops_misc.hip)
bool rope_by_token(const ggml_tensor * dst);

#if defined(__HIPCC__)
// The pair (x0, x1) turned by t = (cos, sin): (x0 cos - x1 sin, x0 sin + x1 cos). A sum of two products may round either of
// them first, as a compiler likes, so what has to give the same bits in several kernels is written out: TOKEN as in the
// kernels that take a token at a time, else as in the one that takes a row
template <bool TOKEN> __device__ __forceinline__ float2 rope_turn(float x0, float x1, float2 t) {
    return make_float2(__builtin_fmaf(x0, t.x, -(x1 * t.y)), TOKEN ? __builtin_fmaf(x0, t.y, x1 * t.x) : __builtin_fmaf(x1, t.x, x0 * t.y));
}

__device__ __forceinline__ void rope_cs(float theta_extrap, const RopeP & p, int i0, float * c, float * s) {
    const float theta_interp = p.freq_scale * theta_extrap;
    float theta = theta_interp;
    float mscale = p.attn_factor;
    if (p.ext_factor != 0.0f) {
        const float y = (i0 / 2 - p.corr0) / fmaxf(0.001f, p.corr1 - p.corr0);
        const float ramp_mix = (1.0f - fminf(1.0f, fmaxf(0.0f, y))) * p.ext_factor;
        theta = theta_interp * (1 - ramp_mix) + theta_extrap * ramp_mix;
        mscale *= 1.0f + 0.1f * logf(1.0f / p.freq_scale);
    }
    *c = cosf(theta) * mscale;
    *s = sinf(theta) * mscale;
}

// Channel pair `ic` of a rotation over several axes (ggml.h GGML_ROPE_TYPE_MROPE / _IMROPE /
// _VISION): the sections' pairs repeat over the head; MROPE gives each axis a run of pairs, IMROPE
// deals them out in turn (pairs beyond an axis' share fall to the fourth), VISION counts each axis'
// exponent from its own first pair. Returns the axis, *e the exponent.
__device__ __forceinline__ int rope_axis(const RopeP & p, int ic, int * e) {
    const int s0 = p.sect[0], s1 = p.sect[1], s2 = p.sect[2], n = s0 + s1 + s2 + p.sect[3];
    const int k = ic % n;
    *e = ic;
    if (p.mode == GGML_ROPE_TYPE_IMROPE) {
        if (k % 3 == 1 && k < 3 * s1) return 1;
        if (k % 3 == 2 && k < 3 * s2) return 2;
        return k % 3 == 0 && k < 3 * s0 ? 0 : 3;
    }
    const int a = k < s0 ? 0 : k < s0 + s1 ? 1 : k < s0 + s1 + s2 ? 2 : 3;
    if (p.mode == GGML_ROPE_TYPE_VISION) *e = k - (a > 0 ? s0 : 0) - (a > 1 ? s1 : 0) - (a > 2 ? s2 : 0);
    return a;
}

// cos and sin (with the sign of the sine) of channel pair ic at position `pos` of its axis. The angle
// in turns, pos * base^(-2e/n_dims) / 2 pi, is formed and reduced to [-1/2, 1/2] in 64 bits: at
// position 30000 a 32-bit product would be off by 1e-3 of a radian. YaRN's interpolation scales the
// frequency, so it enters as a factor.
__device__ __forceinline__ float2 rope_cs_axes(const RopeP & p, int ic, int e, int pos, float ff) {
    double turns = exp2(-2.0 * e / p.n_dims * p.log2_base) * 0.15915494309189535 / (double) ff;
    float mscale = p.attn_factor, mix = 0.0f;
    if (p.ext_factor != 0.0f) {
        const float y = (ic - p.corr0) / fmaxf(0.001f, p.corr1 - p.corr0);
        mix = (1.0f - fminf(1.0f, fmaxf(0.0f, y))) * p.ext_factor;
        mscale *= 1.0f + 0.1f * logf(1.0f / p.freq_scale);
    }
    turns *= (double) p.freq_scale * (1.0 - mix) + mix;
    turns *= pos;
    float s, c;
    sincospif((float) (2.0 * (turns - rint(turns))), &s, &c);
    return make_float2(c * mscale, s * mscale * p.sin_sign);
}

// cos / sin of pair ic of the token whose positions start at pos[t] (n_tok apart by axis), whatever
// the mode: one axis keeps the CPU's recurrence theta_i = pos * scale^i in 32 bits
__device__ __forceinline__ float2 rope_pair(const RopeP & p, int ic, const int32_t * pos, int64_t t, int64_t n_tok, const float * ff) {
    const float f = ff ? ff[ic] : 1.0f;
    if (p.mode & GGML_ROPE_TYPE_MROPE) {
        int e;
        const int a = rope_axis(p, ic, &e);
        return rope_cs_axes(p, ic, e, pos[t + a * n_tok], f);
    }
    float theta = (float) pos[t];
    for (int k = 0; k < ic; ++k) theta *= p.theta_scale;
    float c, s;
    rope_cs(theta / f, p, 2 * ic, &c, &s);
    return make_float2(c, s * p.sin_sign);
}
#endif

}  // namespace mx
