// Forward of the scene attention (scene_attn.h has the mathematics and the layout).
//
// One workgroup: 64 packed rows of one kv head, 16 per wave; K and V tiles of BN keys staged in LDS, the next tile's loads in flight in
// registers while the current one is worked on.  A wave skips 16-key blocks that none of its rows sees, so a tile that holds
// several small scenes costs each wave its own scenes only.
#include "scene_attn.h"

namespace sattn {

// A row whose tile result is not finite, over its visible keys alone: 0 * inf of a masked place must not reach it, while what it does
// see has to come out as the formula says.  One wave; lane l holds columns l and l + 64.
template <typename T> __device__ void row_slow(const SceneAttnArgs &A, int kvh, const RowState &s, int64_t r, int64_t R) {
    const int lane = threadIdx.x & 63;
    const T *q = reinterpret_cast<const T *>(A.q) + s.row * A.q_rs + s.head * A.q_hs;
    const T *k = reinterpret_cast<const T *>(A.k) + kvh * A.k_hs, *v = reinterpret_cast<const T *>(A.v) + kvh * A.v_hs;
    const bool h0 = lane < A.D, h1 = lane + 64 < A.D;
    const float q0 = h0 ? to_f(q[lane]) : 0.f, q1 = h1 ? to_f(q[lane + 64]) : 0.f;
    const float inv_cap = A.cap > 0.f ? 1.f / A.cap : 0.f;
    float m = NEG_INF, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int64_t j = s.lo; j < s.hi; ++j) {
        float raw = (h0 ? q0 * to_f(k[j * A.k_rs + lane]) : 0.f) + (h1 ? q1 * to_f(k[j * A.k_rs + lane + 64]) : 0.f);
        raw = wave_sum(raw);
        const float x = score2(A, raw, inv_cap, s.slope, s.pos, A.kpos + j * A.axes);
        const float mn = fmaxf(m, x), base = mn == NEG_INF ? 0.f : mn;
        const float corr = exp2_(m - base), p = exp2_(x - base);
        l = l * corr + p;
        o0 = o0 * corr + (h0 ? p * to_f(v[j * A.v_rs + lane]) : 0.f);
        o1 = o1 * corr + (h1 ? p * to_f(v[j * A.v_rs + lane + 64]) : 0.f);
        m = mn;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t at = ((int64_t)s.row * A.H + s.head) * A.D;
    T *out = reinterpret_cast<T *>(A.out) + at;
    if (h0) out[lane] = (T)(o0 * inv);
    if (h1) out[lane + 64] = (T)(o1 * inv);
    if (A.o32) {
        if (h0) A.o32[at + lane] = o0 * inv;
        if (h1) A.o32[at + lane + 64] = o1 * inv;
    }
    if (A.lse && lane == 0) A.lse[kvh * R + r] = l == 0.f ? 0.f : m + log2_(l);
}

template <typename T, int DP, int BN>
__global__ __launch_bounds__(256) void scene_attn_fwd_kernel(const SceneAttnArgs A) {
    using X = Tr<T>;
    using L = Tile<T, DP>;
    constexpr int NF = DP / X::KD, NB = BN / 16, DB = DP / 16, PB = X::KB / 16, NC = BN * L::NCH, PER = NC / 256;
    static_assert(NC % 256 == 0 && NB % PB == 0, "tile");
    __shared__ u32x4 sk[NC], sv[NC];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const int kvh = (int)(blockIdx.x % A.KV);
    const int64_t R = (int64_t)A.nq * A.G, r0 = (int64_t)(gridDim.x / A.KV - 1 - blockIdx.x / A.KV) * 64, r = r0 + w * 16 + c;
    const RowState s = row_state(A, kvh, r, R);
    const T *Q = reinterpret_cast<const T *>(A.q) + s.row * A.q_rs + s.head * A.q_hs;
    typename X::frag qf[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) qf[f] = as_frag<T>(load_chunk<T>(Q, f * X::KD + g * X::CH, A.D, A.q_vec));
    // the keys of the workgroup's rows, and of this wave's
    const int qa = (int)(r0 / A.G), qb = (int)((min(r0 + 64, R) - 1) / A.G);
    const int tlo = max(A.row_lo[qa], 0), thi = min(A.row_hi[qb], A.nk);
    const int wlo = __builtin_amdgcn_readfirstlane(__shfl(s.lo, 0)), whi = __builtin_amdgcn_readfirstlane(__shfl(s.hi, 15));
    const int lo_last = __builtin_amdgcn_readfirstlane(__shfl(s.lo, 15)), hi_first = __builtin_amdgcn_readfirstlane(__shfl(s.hi, 0));
    const T *K = reinterpret_cast<const T *>(A.k) + kvh * A.k_hs, *V = reinterpret_cast<const T *>(A.v) + kvh * A.v_hs;
    const float inv_cap = A.cap > 0.f ? 1.f / A.cap : 0.f;

    u32x4 rk[PER], rv[PER];
    auto fetch = [&](int kb) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = tid + i * 256, key = kb + e / L::NCH, ch = e % L::NCH;
            const u32x4 z = {0u, 0u, 0u, 0u};
            const bool in = key < thi;
            rk[i] = in ? load_chunk<T>(K + (int64_t)key * A.k_rs, ch * X::CH, A.D, A.k_vec) : z;
            rv[i] = in ? load_chunk<T>(V + (int64_t)key * A.v_rs, ch * X::CH, A.D, A.v_vec) : z;
        }
    };
    f32x4 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = NEG_INF, l = 0.f;
    if (tlo < thi) fetch(tlo);
    for (int kb = tlo; kb < thi; kb += BN) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = tid + i * 256;
            sk[L::slot(e / L::NCH, e % L::NCH)] = rk[i];
            sv[L::slot(e / L::NCH, e % L::NCH)] = rv[i];
        }
        __syncthreads();
        if (kb + BN < thi) fetch(kb + BN);
        if (kb >= whi || kb + BN <= wlo) continue;          // the barriers above are met by every wave of the next round
        f32x4 x[NB];
        float top = NEG_INF;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int k0 = kb + b * 16;
            x[b] = f32x4{NEG_INF, NEG_INF, NEG_INF, NEG_INF};
            if (k0 >= whi || k0 + 16 <= wlo) continue;
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < NF; ++f) a = mma(frag_rows<T, DP>(sk, b * 16, f, lane), qf[f], a);
            const bool masked = k0 < lo_last || k0 + 16 > hi_first;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = k0 + 4 * g + i;
                const float y = score2(A, a[i], inv_cap, s.slope, s.pos, A.kpos + (int64_t)min(key, A.nk - 1) * A.axes);
                x[b][i] = masked && (key < s.lo || key >= s.hi) ? NEG_INF : y;
                top = fmaxf(top, x[b][i]);
            }
        }
        top = fmaxf(group_max(top), m);
        const float base = top == NEG_INF ? 0.f : top, corr = exp2_(m - base);
        m = top;
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[b][i] = exp2_(x[b][i] - base);
                sum += x[b][i];
            }
        l = l * corr + sum;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] *= corr;
#pragma unroll
        for (int j = 0; j < NB / PB; ++j) {
            const int k0 = kb + j * X::KB;
            if (k0 >= whi || k0 + X::KB <= wlo) continue;
            const typename X::frag p = pack_p(x + j * PB, T());
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] = mma(frag_cols<DP>(sv, j * X::KB, d, lane, T()), p, o[d]);
        }
    }
    l = group_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bool fine = finite_(l);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[d][i] *= inv;
            fine = fine && finite_(o[d][i]);
        }
    if (r < R) {
        const int64_t at = ((int64_t)s.row * A.H + s.head) * A.D;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            store4(reinterpret_cast<T *>(A.out) + at, o[d], d * 16 + g * 4, A.D, A.o_vec != 0);
            if (A.o32) store4(A.o32 + at, o[d], d * 16 + g * 4, A.D, A.o_vec != 0);
        }
        if (A.lse && g == 0) A.lse[kvh * R + r] = l == 0.f ? 0.f : m + log2_(l);
    }
    uint64_t bad = __ballot(!fine && r < R);
    while (bad) {                                           // wave-uniform; the same row may be named by several lane groups
        const int src = __builtin_ctzll(bad) & 15;
        bad &= ~(0x0001000100010001ull << src);
        RowState t = row_state(A, kvh, r0 + w * 16 + src, R);
        row_slow<T>(A, kvh, t, r0 + w * 16 + src, R);
    }
}

template <typename T, int DP, int BN> hipError_t launch_fwd(const SceneAttnArgs &A, hipStream_t st) {
    const int64_t tiles = ((int64_t)A.nq * A.G + 63) / 64;
    hipLaunchKernelGGL((scene_attn_fwd_kernel<T, DP, BN>), dim3((unsigned)(tiles * A.KV)), dim3(256), 0, st, A);
    return hipGetLastError();
}

}  // namespace sattn

extern "C" hipError_t dn_scene_attn_fwd(const SceneAttnArgs *A, int bf, hipStream_t st) {
    using namespace sattn;
    const int D = A->D;
    if (bf) return D <= 32 ? launch_fwd<bf16, 32, 64>(*A, st) : D <= 64 ? launch_fwd<bf16, 64, 64>(*A, st) : launch_fwd<bf16, 128, 64>(*A, st);
    return D <= 16 ? launch_fwd<float, 16, 64>(*A, st) : D <= 32 ? launch_fwd<float, 32, 64>(*A, st) : D <= 64 ? launch_fwd<float, 64, 64>(*A, st)
                                                                                              : launch_fwd<float, 128, 32>(*A, st);
}
