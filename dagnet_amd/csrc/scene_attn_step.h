// Arguments of the step kernel (scene_attn_step.hip), shared with the C entry.
#pragma once
#include "scene_attn.h"

struct SceneStepArgs {
    SceneAttnArgs a;                 // nk, row and key bounds unused
    const int32_t *q_ptr, *k_len;    // [scenes + 1], [scenes]
    int64_t k_ss, v_ss;              // element strides of scenes in the cache
    int32_t scenes, room, splits, cblocks;     // cblocks: blocks of 16 packed rows a scene
    float *part, *stat;              // splits > 1: [nq * H][splits][D], [nq * H][splits][2]
};
