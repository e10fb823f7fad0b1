// Arguments of the rotary kernel (rotary.hip), shared with the C entry.
#pragma once
#include <stdint.h>

struct RotaryArgs {
    const void *q, *k, *pos;
    void *qo, *ko;
    const double *turns;             // [pairs]: frequency / 2 pi
    const int32_t *axis;             // [pairs]
    int64_t n, q_rs, q_hs, k_rs, k_hs, qo_rs, qo_hs, ko_rs, ko_hs;
    int32_t hq, hk, D, pairs, axes, interleaved, rows_per;
    float sign;
};
