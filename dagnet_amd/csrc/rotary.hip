// Rotary positions with several axes: pair i of a head's columns is turned by the angle pos[axis(i)] * freq(i),
//     (a, b) -> (a cos - b sin, b cos + a sin),       backward: the same turn by the opposite angle.
// Pairs stand side by side (interleaved: columns 2 i, 2 i + 1) or half a turned width apart (columns i, P + i); columns behind the 2 P
// turned ones pass through.
//
// The angle is taken in turns and in fp64 (freq / 2 pi comes as a double): a time stamp of 10^6 times a frequency near 1 has lost
// its sine in fp32.  What is left of the turn after rint() goes through sincospi in fp32.  A workgroup computes the sines of its rows once into
// LDS and applies them to all heads of q and k, so the kernel moves the data once and is bound by memory.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "rotary.h"

namespace rot {

typedef __bf16 bf16;

constexpr int ROWS_MAX = 16;

template <typename T> __device__ __forceinline__ float ld(const T *p) { return (float)*p; }

template <typename T, typename P>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs A) {
    extern __shared__ float2 cs[];                       // [rows][pairs]
    const int64_t row0 = (int64_t)blockIdx.x * A.rows_per;
    const int rows = (int)min((int64_t)A.rows_per, A.n - row0);
    for (int e = threadIdx.x; e < rows * A.pairs; e += 256) {
        const int r = e / A.pairs, i = e - r * A.pairs;
        const double t = (double)reinterpret_cast<const P *>(A.pos)[(row0 + r) * A.axes + A.axis[i]] * A.turns[i];
        const float f = (float)(t - rint(t));
        float s, c;
        sincospif(2.f * f, &s, &c);
        cs[e] = float2{c, A.sign * s};
    }
    __syncthreads();
    const int heads = A.hq + A.hk, D = A.D, half = (D + 1) / 2;
    // work item: one pair of columns (or up to two columns that pass through) of one head of one row
    for (int e = threadIdx.x; e < rows * heads * half; e += 256) {
        const int r = e / (heads * half), h = (e / half) % heads, i = e % half;
        const int64_t row = row0 + r;
        const bool isq = h < A.hq;
        const T *x = reinterpret_cast<const T *>(isq ? A.q : A.k) + (isq ? row * A.q_rs + h * A.q_hs : row * A.k_rs + (h - A.hq) * A.k_hs);
        T *y = reinterpret_cast<T *>(isq ? A.qo : A.ko) + (isq ? row * A.qo_rs + h * A.qo_hs : row * A.ko_rs + (h - A.hq) * A.ko_hs);
        if (i < A.pairs) {
            const int ia = A.interleaved ? 2 * i : i, ib = A.interleaved ? 2 * i + 1 : A.pairs + i;
            const float2 v = cs[r * A.pairs + i];
            const float a = ld(x + ia), b = ld(x + ib);
            y[ia] = (T)(a * v.x - b * v.y);
            y[ib] = (T)(b * v.x + a * v.y);
        } else {
            y[2 * i] = x[2 * i];
            if (2 * i + 1 < D) y[2 * i + 1] = x[2 * i + 1];
        }
    }
}

template <typename T> hipError_t launch(const RotaryArgs &A, int pos_type, hipStream_t st) {
    const unsigned blocks = (unsigned)((A.n + A.rows_per - 1) / A.rows_per);
    const size_t lds = sizeof(float2) * A.rows_per * A.pairs;
    if (pos_type == 0) hipLaunchKernelGGL((rotary_kernel<T, float>), dim3(blocks), dim3(256), lds, st, A);
    else if (pos_type == 1) hipLaunchKernelGGL((rotary_kernel<T, int32_t>), dim3(blocks), dim3(256), lds, st, A);
    else hipLaunchKernelGGL((rotary_kernel<T, int64_t>), dim3(blocks), dim3(256), lds, st, A);
    return hipGetLastError();
}

}  // namespace rot

extern "C" hipError_t dn_rotary(const RotaryArgs *A, int bf, int pos_type, hipStream_t st) {
    RotaryArgs B = *A;
    B.rows_per = rot::ROWS_MAX;
    return bf ? rot::launch<rot::bf16>(B, pos_type, st) : rot::launch<float>(B, pos_type, st);
}
