// tc_step.hpp -- arguments and launchers of the operators around a step's products and
// attention (tc_plan.hip, tc_rope.hip, tc_norm.hip, tc_logits.hip).
#pragma once

#include "tc_attn_common.hpp"
#include "tc_step.h"

namespace tc {

constexpr uint32_t kPlanMost = 1u << 30;       // sums of pages are held to this
constexpr int32_t kLenMost = 0x7FFFFFFF - 64;  // tokens of a sequence

hipError_t launch_plan(const tc_plan &p, hipStream_t st);

// Rotation as the kernels take it.
struct RopeArgs {
    const double *turns;
    uint32_t n_rot, half;  // half of n_rot
    int32_t layout;
    float factor;
};
// Heads of one kind in a token's row.
struct RopeHeads {
    const void *x;
    uint64_t stride;  // elements between tokens
    uint32_t heads;
    const float *norm;  // weights of the heads' norm, null: none
};
struct RopeCall {
    KvArgs kv;  // tokens and, with a cache, batch (without: n_tokens and dim only)
    RopeArgs rope;
    RopeHeads q, k, v;
    void *q_out;
    uint64_t q_out_stride;
    const int32_t *position;  // of each row where there is no batch
    float eps;
    int xtype;
};
constexpr uint32_t kRopeUnits = 4;  // heads of a lane in long calls
// Lanes that have a head between them.
inline uint32_t rope_lane_log(uint32_t dim) {
    uint32_t log = 1;
    while ((16u << (log - 1)) < dim) ++log;
    return log;
}
hipError_t launch_rope_kv(const RopeCall &c, int ctype, hipStream_t st);
hipError_t launch_rope_rows(const RopeCall &c, hipStream_t st);
// Turns of pair i: theta^(-2i / n_rot) / 2 pi, changed as the kind says; first, ramp: where
// YARN's ramp begins and how long it is.
struct TurnsCall {
    int32_t kind;
    uint32_t n_rot;
    double theta, factor, original, low, high, first, ramp;
    const float *divisors;
    double *turns;
};
hipError_t launch_rope_turns(const TurnsCall &c, hipStream_t st);

// A norm as the kernel takes it.
struct NormArgs {
    const float *weight, *bias;
    float eps, offset;
    int32_t kind;  // -1: none
};
struct NormCall {
    uint32_t rows, cols;
    const void *h, *y, *gate;
    void *h_out, *x;
    int32_t h_type, y_type, x_type, gate_type, gate_kind, gate_sigmoid;
    uint64_t h_stride, y_stride, h_out_stride, x_stride;
    NormArgs post, pre;
    float scale;
    // quantized activations (act_layout), null: none
    int8_t *qs;
    float *d;
    int16_t *bsums;
    uint16_t *dg;
    int32_t act_q8_0;  // 32-wide blocks instead of 256-wide ones
    // (set by the launcher) 1 / cols, the power of two at it or below, their quotient
    float inv_cols, down, inv_cols_down;
};
hipError_t launch_norm(const NormCall &c, int num_cu, hipStream_t st);

struct LogitCall {
    tc_logit_rules r;
    const void *logits;
    float *out;
    uint64_t x_stride, out_stride;
    int32_t xtype;
    uint32_t vocab, n_seq, n_tokens;
    const int32_t *start, *tokens;
};
hipError_t launch_logits(const LogitCall &c, int num_cu, hipStream_t st);

}  // namespace tc
