// Rotary positions with several axes: pair i of a head's columns is turned by the angle pos[axis(i)] * freq(i),
//     (a, b) -> (a cos - b sin, b cos + a sin),       backward: the same turn by the opposite angle.
// Pairs stand side by side (interleaved: columns 2 i, 2 i + 1) or half a turned width apart (columns i, P + i); columns behind the 2 P
// turned ones pass through.
//
// The angle is taken in turns and in fp64 (freq / 2 pi comes as a double): a time stamp of 10^6 times a frequency near 1 has lost
// its sine in fp32.  What is left of the turn after rint() goes through sincospi in fp32.  A workgroup computes the sines of its rows once into
// LDS and applies them to all heads of q and k, so the kernel moves the data once and is bound by memory: a thread owns one place of a
// row (a head's 16-byte chunk with its partner chunk) and walks the workgroup's rows, four rows' loads in flight.
// Measured: 65 521 bf16 rows of 16 and 4 heads of 128, forward and backward 259 us for 1343 MB, 5.2 TB/s.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "rotary.h"

namespace rot {

typedef __bf16 bf16;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T, int VE> struct Vec { T e[VE]; };
template <typename T, int VE> __device__ __forceinline__ Vec<T, VE> ld(const T *p) {
    if constexpr (VE * sizeof(T) == 16) {
        union { u32x4 u; Vec<T, VE> v; } x;
        x.u = *reinterpret_cast<const u32x4 *>(p);
        return x.v;
    } else return *reinterpret_cast<const Vec<T, VE> *>(p);
}
template <typename T, int VE> __device__ __forceinline__ void st(T *p, Vec<T, VE> v) {
    if constexpr (VE * sizeof(T) == 16) {
        union { u32x4 u; Vec<T, VE> v; } x;
        x.v = v;
        *reinterpret_cast<u32x4 *>(p) = x.u;
    } else *reinterpret_cast<Vec<T, VE> *>(p) = v;
}

// VE: columns a thread handles at a time (16 bytes where widths and strides allow it, else 1).  An item is
//   halves: VE pairs = columns i .. and P + i ..;   interleaved: VE pairs = 2 VE columns from 2 i;   behind the pairs: up to 2 VE columns that pass.
template <typename T, typename P, int VE>
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
    const int D = A.D, turned = A.pairs / VE, items = turned + (D - 2 * A.pairs + 2 * VE - 1) / (2 * VE), per_row = items * (A.hq + A.hk);
    const int lanes = per_row < 256 ? 256 / per_row : 1;              // rows side by side
    const int sub = per_row < 256 ? threadIdx.x / per_row : 0;
    if (sub >= lanes) return;
    for (int e = per_row < 256 ? threadIdx.x % per_row : threadIdx.x; e < per_row; e += 256) {
        const int h = e / items, i = e - h * items;
        const bool isq = h < A.hq;
        const T *x = isq ? reinterpret_cast<const T *>(A.q) + h * A.q_hs : reinterpret_cast<const T *>(A.k) + (h - A.hq) * A.k_hs;
        T *y = isq ? reinterpret_cast<T *>(A.qo) + h * A.qo_hs : reinterpret_cast<T *>(A.ko) + (h - A.hq) * A.ko_hs;
        const int64_t xs = isq ? A.q_rs : A.k_rs, ys = isq ? A.qo_rs : A.ko_rs;
        const bool pass = i >= turned;
        const int ca = pass ? 2 * A.pairs + (i - turned) * 2 * VE : A.interleaved ? 2 * i * VE : i * VE;
        const int cb = pass || A.interleaved ? ca + VE : A.pairs + ca;
        const bool two = cb < D;                                       // an odd width's last column stands alone
        constexpr int U = 4;
        for (int r = sub; r < rows; r += U * lanes) {
            Vec<T, VE> a[U], b[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int rr = min(r + u * lanes, rows - 1);
                const T *p = x + (row0 + rr) * xs;
                a[u] = ld<T, VE>(p + ca);
                b[u] = ld<T, VE>(p + (two ? cb : ca));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int rr = r + u * lanes;
                if (rr >= rows) break;
                if (!pass) {
                    const float2 *t = cs + rr * A.pairs + i * VE;
                    if (A.interleaved) {
#pragma unroll
                        for (int j = 0; j < VE; ++j) {
                            // pair j of the item: elements 2 j, 2 j + 1 of (a, b); VE 1: a and b themselves
                            T &ea = VE == 1 ? a[u].e[0] : (2 * j < VE ? a[u].e[(2 * j) % VE] : b[u].e[(2 * j) % VE]);
                            T &eb = VE == 1 ? b[u].e[0] : (2 * j < VE ? a[u].e[(2 * j + 1) % VE] : b[u].e[(2 * j + 1) % VE]);
                            const float fa = (float)ea, fb = (float)eb;
                            ea = (T)(fa * t[j].x - fb * t[j].y);
                            eb = (T)(fb * t[j].x + fa * t[j].y);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < VE; ++j) {
                            const float fa = (float)a[u].e[j], fb = (float)b[u].e[j];
                            a[u].e[j] = (T)(fa * t[j].x - fb * t[j].y);
                            b[u].e[j] = (T)(fb * t[j].x + fa * t[j].y);
                        }
                    }
                }
                T *p = y + (row0 + rr) * ys;
                st<T, VE>(p + ca, a[u]);
                if (two) st<T, VE>(p + cb, b[u]);
            }
        }
    }
}

template <typename T, typename P> hipError_t launch(const RotaryArgs &A, hipStream_t st) {
    constexpr int VE = 16 / sizeof(T);
    const unsigned blocks = (unsigned)((A.n + A.rows_per - 1) / A.rows_per);
    const size_t lds = sizeof(float2) * A.rows_per * A.pairs;
    // whole chunks on both sides of a pair, and what passes through in whole chunks too
    const int s = (int)sizeof(T);
    auto fits = [&](const void *p, int64_t rs, int64_t hs) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && rs * s % 16 == 0 && hs * s % 16 == 0; };
    const bool wide = A.pairs % VE == 0 && A.D % VE == 0 && fits(A.q, A.q_rs, A.q_hs) && fits(A.qo, A.qo_rs, A.qo_hs) &&
                      (A.hk == 0 || (fits(A.k, A.k_rs, A.k_hs) && fits(A.ko, A.ko_rs, A.ko_hs)));
    if (wide) hipLaunchKernelGGL((rotary_kernel<T, P, VE>), dim3(blocks), dim3(256), lds, st, A);
    else hipLaunchKernelGGL((rotary_kernel<T, P, 1>), dim3(blocks), dim3(256), lds, st, A);
    return hipGetLastError();
}

}  // namespace rot

extern "C" hipError_t dn_rotary(const RotaryArgs *A, int bf, int pos_type, hipStream_t st) {
    RotaryArgs B = *A;
    // 16 rows a workgroup (their sines fit 64 KB of LDS up to 512 pairs), fewer where that would leave CUs without work
    const int64_t per = A->n / 1024;
    B.rows_per = per >= 16 ? 16 : per >= 1 ? (int)per : 1;
    if (bf) return pos_type == 0 ? rot::launch<rot::bf16, float>(B, st) : pos_type == 1 ? rot::launch<rot::bf16, int32_t>(B, st) : rot::launch<rot::bf16, int64_t>(B, st);
    return pos_type == 0 ? rot::launch<float, float>(B, st) : pos_type == 1 ? rot::launch<float, int32_t>(B, st) : rot::launch<float, int64_t>(B, st);
}
