// Scene attention of the new rows of a step over kept keys (scene_attn.h has the mathematics and the layout): scene s keeps its keys and
// values in rows 0 .. k_len[s] - 1 of its own stretch of a cache, and all of its new rows see all of them.
//
// Few rows, many keys: the keys are read once and bound the kernel.  One workgroup takes one scene, one kv head, 16 packed rows (the new
// rows times the heads that share keys) and one split of the keys; its four waves take 32 (16-bit) or 16 (fp32) keys in turn, K straight
// from memory into the first product's operand, V through a wave's own stretch of LDS for the transposed one.  The splits' partial
// outputs, maxima and sums meet in scene_attn_join_kernel.
#include "scene_attn.h"
#include "scene_attn_step.h"
#include <algorithm>

namespace sattn {

template <typename T, int DP> __global__ __launch_bounds__(256) void scene_attn_step_kernel(const SceneStepArgs A) {
    using X = Tr<T>;
    using L = Tile<T, DP>;
    constexpr int NF = DP / X::KD, DB = DP / 16, PB = X::KB / 16, NC = X::KB * L::NCH, PER = NC / 64;
    static_assert(NC % 64 == 0, "tile");
    __shared__ u32x4 sv[4][NC];
    __shared__ float sm[4][16], sl[4][16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    int64_t id = blockIdx.x;
    const int cb = (int)(id % A.cblocks);
    id /= A.cblocks;
    const int split = (int)(id % A.splits);
    id /= A.splits;
    const int kvh = (int)(id % A.a.KV), sc = (int)(id / A.a.KV);
    const int q0 = max(A.q_ptr[sc], 0), q1 = min(A.q_ptr[sc + 1], A.a.nq);
    const int64_t n = (int64_t)(q1 - q0) * A.a.G;
    if (cb * 16 >= n) return;                                       // the whole workgroup
    const int64_t pr = min((int64_t)cb * 16 + c, n - 1);
    const int row = q0 + (int)(pr / A.a.G), head = kvh * A.a.G + (int)(pr % A.a.G);
    const int len = min(max(A.k_len[sc], 0), A.room);
    const int per = (int)((((int64_t)len + A.splits - 1) / A.splits + 4 * X::KB - 1) / (4 * X::KB)) * (4 * X::KB);   // whole rounds of the four waves
    const int ka = (int)min((int64_t)split * per, (int64_t)len), kz = (int)min((int64_t)ka + per, (int64_t)len);
    const float slope2 = A.a.axes ? A.a.slopes[head] * LOG2E : 0.f, inv_cap = A.a.cap > 0.f ? 1.f / A.a.cap : 0.f;
    float qpos[3] = {0.f, 0.f, 0.f};
    for (int a = 0; a < A.a.axes; ++a) qpos[a] = A.a.qpos[(int64_t)row * A.a.axes + a];
    const T *Q = reinterpret_cast<const T *>(A.a.q) + row * A.a.q_rs + head * A.a.q_hs;
    const T *K = reinterpret_cast<const T *>(A.a.k) + sc * A.k_ss + kvh * A.a.k_hs, *V = reinterpret_cast<const T *>(A.a.v) + sc * A.v_ss + kvh * A.a.v_hs;
    const float *kpos = A.a.kpos + (int64_t)sc * A.room * A.a.axes;
    typename X::frag qf[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) qf[f] = as_frag<T>(load_chunk<T>(Q, f * X::KD + g * X::CH, A.a.D, A.a.q_vec));

    u32x4 rk[PB][NF], rv[PER];
    auto fetch = [&](int k0) {                                      // keys behind the last one stand in as the last one, masked below
#pragma unroll
        for (int b = 0; b < PB; ++b) {
            const T *p = K + (int64_t)min(k0 + b * 16 + c, len - 1) * A.a.k_rs;
#pragma unroll
            for (int f = 0; f < NF; ++f) rk[b][f] = load_chunk<T>(p, f * X::KD + g * X::CH, A.a.D, A.a.k_vec);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane + i * 64;
            rv[i] = load_chunk<T>(V + (int64_t)min(k0 + e / L::NCH, len - 1) * A.a.v_rs, (e % L::NCH) * X::CH, A.a.D, A.a.v_vec);
        }
    };
    f32x4 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = NEG_INF, l = 0.f;
    int k0 = ka + w * X::KB;
    if (k0 < kz) fetch(k0);
    for (; k0 < kz; k0 += 4 * X::KB) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane + i * 64;
            sv[w][L::slot(e / L::NCH, e % L::NCH)] = rv[i];
        }
        f32x4 x[PB];
        float top = NEG_INF;
#pragma unroll
        for (int b = 0; b < PB; ++b) {
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < NF; ++f) a = mma(as_frag<T>(rk[b][f]), qf[f], a);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = k0 + b * 16 + 4 * g + i;
                const float y = score2(A.a, a[i], inv_cap, slope2, qpos, kpos + (int64_t)min(key, len - 1) * A.a.axes);
                x[b][i] = key < kz ? y : NEG_INF;
                top = fmaxf(top, x[b][i]);
            }
        }
        if (k0 + 4 * X::KB < kz) fetch(k0 + 4 * X::KB);
        top = fmaxf(group_max(top), m);
        const float base = top == NEG_INF ? 0.f : top, corr = exp2_(m - base);
        m = top;
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < PB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[b][i] = exp2_(x[b][i] - base);
                sum += x[b][i];
            }
        l = l * corr + sum;
        const typename X::frag p = pack_p(x, T());
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");      // the wave's own LDS writes, before its transposed reads
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = mma(frag_cols<DP>(sv[w], 0, d, lane, T()), p, o[d] * corr);
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    l = group_sum(l);
    // the four waves' parts: statistics first, then the outputs, rescaled, through the waves' V stretches
    if (g == 0) { sm[w][c] = m; sl[w][c] = l; }
    __syncthreads();
    float M = NEG_INF, Lsum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) M = fmaxf(M, sm[i][c]);
    const float base = M == NEG_INF ? 0.f : M;
#pragma unroll
    for (int i = 0; i < 4; ++i) Lsum += sl[i][c] * exp2_(sm[i][c] - base);
    const float corr = exp2_(m - base);
    // [16][DP] floats a wave
    float *so = reinterpret_cast<float *>(&sv[0][0]);
    constexpr int CAPF = 4 * NC * 4 / 16;                            // floats of LDS per row
    constexpr int WAVES = CAPF >= 4 * DP ? 4 : CAPF / DP;            // waves whose outputs fit at once
    static_assert(WAVES >= 1, "LDS");
    f32x4 acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w0 = 0; w0 < 4; w0 += WAVES) {
        if (w >= w0 && w < w0 + WAVES) {
#pragma unroll
            for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4 *>(so + ((w - w0) * 16 + c) * DP + d * 16 + g * 4) = o[d] * corr;
        }
        __syncthreads();
        if (w == 0) {
#pragma unroll
            for (int i = 0; i < WAVES; ++i)
                if (w0 + i < 4)
#pragma unroll
                    for (int d = 0; d < DB; ++d) acc[d] += *reinterpret_cast<const f32x4 *>(so + (i * 16 + c) * DP + d * 16 + g * 4);
        }
        __syncthreads();
    }
    if (w != 0 || (int64_t)cb * 16 + c >= n) return;
    const int64_t item = (int64_t)row * A.a.H + head;
    if (A.splits == 1) {
        const float inv = Lsum == 0.f ? 0.f : 1.f / Lsum;
#pragma unroll
        for (int d = 0; d < DB; ++d) store4(reinterpret_cast<T *>(A.a.out) + item * A.a.D, acc[d] * inv, d * 16 + g * 4, A.a.D, A.a.o_vec != 0);
        return;
    }
    float *part = A.part + (item * A.splits + split) * A.a.D;
#pragma unroll
    for (int d = 0; d < DB; ++d) store4(part, acc[d], d * 16 + g * 4, A.a.D, A.a.D % 4 == 0);
    if (g == 0) {
        A.stat[(item * A.splits + split) * 2] = M;
        A.stat[(item * A.splits + split) * 2 + 1] = Lsum;
    }
}

// one wave per (row, head)
template <typename T> __global__ __launch_bounds__(256) void scene_attn_join_kernel(const SceneStepArgs A) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= (int64_t)A.a.nq * A.a.H) return;
    const float *stat = A.stat + item * A.splits * 2, *part = A.part + item * A.splits * A.a.D;
    float M = NEG_INF;
    for (int i = 0; i < A.splits; ++i) M = fmaxf(M, stat[2 * i]);
    const float base = M == NEG_INF ? 0.f : M;
    float l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int i = 0; i < A.splits; ++i) {
        const float f = exp2_(stat[2 * i] - base);
        l += f * stat[2 * i + 1];
        if (lane < A.a.D) o0 += f * part[(int64_t)i * A.a.D + lane];
        if (lane + 64 < A.a.D) o1 += f * part[(int64_t)i * A.a.D + lane + 64];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *out = reinterpret_cast<T *>(A.a.out) + item * A.a.D;
    if (lane < A.a.D) out[lane] = (T)(o0 * inv);
    if (lane + 64 < A.a.D) out[lane + 64] = (T)(o1 * inv);
}

template <typename T, int DP> hipError_t launch_step(const SceneStepArgs &A, hipStream_t st) {
    const int64_t blocks = (int64_t)A.scenes * A.a.KV * A.splits * A.cblocks;
    hipLaunchKernelGGL((scene_attn_step_kernel<T, DP>), dim3((unsigned)blocks), dim3(256), 0, st, A);
    if (A.splits > 1) hipLaunchKernelGGL((scene_attn_join_kernel<T>), dim3((unsigned)(((int64_t)A.a.nq * A.a.H + 3) / 4)), dim3(256), 0, st, A);
    return hipGetLastError();
}

}  // namespace sattn

extern "C" hipError_t dn_scene_attn_step(const SceneStepArgs *A, int bf, hipStream_t st) {
    using namespace sattn;
    const int D = A->a.D;
    if (bf) return D <= 32 ? launch_step<bf16, 32>(*A, st) : D <= 64 ? launch_step<bf16, 64>(*A, st) : launch_step<bf16, 128>(*A, st);
    return D <= 16 ? launch_step<float, 16>(*A, st) : D <= 32 ? launch_step<float, 32>(*A, st) : D <= 64 ? launch_step<float, 64>(*A, st) : launch_step<float, 128>(*A, st);
}

// Splits of the keys: a multiple of the chip's 256 CUs in workgroups (four to a CU), but no split below 256 keys of the cache.
extern "C" int dn_scene_attn_step_splits(int64_t groups, int room) {
    const int64_t want = (1024 + groups - 1) / groups, most = (room + 255) / 256;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 64));
}
