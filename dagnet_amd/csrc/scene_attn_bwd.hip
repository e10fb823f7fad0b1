// Backward of the scene attention (scene_attn.h has the mathematics and the layout).
//     p_ij = 2^(x_ij - lse_i),  dp_ij = do_i.v_j,  ds_ij = p_ij (dp_ij - delta_i),  delta_i = do_i.o_i
//     dslope_h = - sum_ij ds_ij |pos_i - pos_j|;   dz_ij = ds_ij (1 - tanh^2) scale;   dq_i = sum_j dz_ij k_j,  dk_j = sum_i dz_ij q_i,
//     dv_j = sum_i p_ij do_i
// Two kernels recompute p from the saved lse, one with query rows on the lanes' columns (dq, dslope), one with keys on them (dk, dv): every
// sum has one owner and one order, so results repeat bit for bit.
// delta is taken from the unrounded output.  What is left of its error (in bf16 the forward's p was rounded for its second product) moves
// every ds of a row by p_ij e_i.  dslope, a sum over all scores of which most cancels, does not forgive that, but a row's ds have to
// add up to nothing, so e_i = - sum_j ds_ij is known and what it did to dslope is taken back: three sums per row instead of one.
// lse_i = m + log2 l is one fp32 number: its rounding, half an ulp, scales all p of a row alike (fp32, 4096 scenes of ten rows: results and gradients together
// 2.6e-7 from the 64-bit formulas).  bf16: dz (dq) and p and dz (dk, dv) are rounded once each for their products; results and gradients together are off by 0.24 %,
// their own rounding alone by 0.17.
//
// By counters: with a cap and three axes bound by vector instructions (48 and 50 a visible score, issuing in 72 and 68 % of the CUs' busy clocks); without either, 96
// wide, as much by LDS (51 - 53 % of the clocks, half of them bank conflicts; vector 36 - 39 %, matrix 23 - 26 %).  Measured: 4093 causal bf16 rows of 8 heads of 96 to 2, dq 81 us
// (6 D operations a pair: 476 TFLOP/s), dk and dv 118 us (8 D: 436), joins 9 us each; 32 scenes of 500 bf16 rows, 8 heads of 64, cap and three axes, 85 and
// 93 us; 4096 fp32 scenes of ten rows, 4 heads of 16, 32 us each.  One block of 16 rows (or keys) a wave: two of 128 columns would keep 192 registers of sums
// and operands before the first score.
#include "scene_attn.h"

namespace sattn {

// One chunk of columns of delta = sum_d do o; lane group g of a row takes the chunks at g CH, KD + g CH, .., in this order in both kernels, so that
// a gradient does not depend on which others are wanted.
template <typename T> __device__ __forceinline__ float delta_chunk(float sum, const float *o, typename Tr<T>::frag gf, int d, int D, int vec) {
#pragma unroll
    for (int i = 0; i < Tr<T>::CH; i += 4) {
        const f32x4 v = __builtin_bit_cast(f32x4, load_chunk<float>(o, d + i, D, vec));
#pragma unroll
        for (int j = 0; j < 4; ++j) sum = fmaf(d + i + j < D ? v[j] : 0.f, d + i + j < D ? to_f(gf[i + j]) : 0.f, sum);
    }
    return sum;
}

// delta[kvh][row G + g], a (row, head) pair to four lanes.  Only where dq is not wanted: the dq kernel has do in registers and computes it on the way.
template <typename T> __global__ __launch_bounds__(256) void scene_attn_delta_kernel(const SceneAttnArgs A) {
    const int64_t n = (int64_t)A.nq * A.H, i = (int64_t)blockIdx.x * 64 + (threadIdx.x >> 2);
    const int part = threadIdx.x & 3;
    const int64_t row = min(i, n - 1) / A.H;
    const int head = (int)(min(i, n - 1) - row * A.H), kvh = head / A.G;
    const T *g = reinterpret_cast<const T *>(A.dout) + row * A.do_rs + head * A.do_hs;
    const float *o = A.o32 + (row * A.H + head) * A.D;
    float s = 0.f;
    for (int d = part * Tr<T>::CH; d < A.D; d += Tr<T>::KD) s = delta_chunk<T>(s, o, as_frag<T>(load_chunk<T>(g, d, A.D, A.do_vec)), d, A.D, A.o32_vec);
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    if (i < n && part == 0) A.delta[(int64_t)kvh * A.nq * A.G + row * A.G + (head - kvh * A.G)] = s;
}

// dslopes[h] = sum over the rows of what the dq kernel left per packed row; one workgroup per head, fp64, fixed order, 16 loads a thread in
// flight (a workgroup alone is bound by their latency)
static __global__ __launch_bounds__(1024) void scene_attn_dslope_kernel(int nq, int G, const float *__restrict__ part, float *__restrict__ out) {
    __shared__ double sh[16];
    const int h = blockIdx.x, kvh = h / G, g = h - kvh * G;
    const float *p = part + (int64_t)kvh * nq * G + g;
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < nq; i += 16384) {
        float v[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) v[u] = p[min(i + u * 1024, (int64_t)nq - 1) * G];
#pragma unroll
        for (int u = 0; u < 16; ++u) s += i + u * 1024 < nq ? v[u] : 0.f;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) s += sh[i];
        out[h] = (float)s;
    }
}

struct Grad { float p, ds, dz, dist; };     // dz without the factor scale

// p, ds and dz of one pair from the raw products
__device__ __forceinline__ Grad pair_grad(const SceneAttnArgs &A, float raw, float dp, float inv_cap, float slope2, const float *qpos,
                                          const float *kpos, float lse, float delta) {
    Grad r;
    float x = raw * A.scale, t = 0.f;
    if (A.cap > 0.f) {
        t = tanh_(x * inv_cap);
        x = A.cap * t;
    }
    x *= LOG2E;
    r.dist = 0.f;
    if (A.axes) {
        r.dist = distance(A.axes, qpos, kpos);
        x -= slope2 * r.dist;
    }
    r.p = exp2_(x - lse);
    r.ds = r.p * (dp - delta);
    r.dz = A.cap > 0.f ? r.ds * (1.f - t * t) : r.ds;
    return r;
}

// a row's part of dslope: sums of ds, ds dist and p dist, the delta's error taken back (above)
struct Slope {
    double ds = 0.0, dsd = 0.0, pd = 0.0;
    __device__ __forceinline__ void add(const Grad &g) {
        ds += g.ds;
        dsd += g.ds * g.dist;
        pd += g.p * g.dist;
    }
    __device__ __forceinline__ float row() const { return (float)(ds * pd - dsd); }
    __device__ __forceinline__ void over_groups() {                               // the four lane groups of a row together
        ds += __shfl_xor(ds, 16);   ds += __shfl_xor(ds, 32);
        dsd += __shfl_xor(dsd, 16); dsd += __shfl_xor(dsd, 32);
        pd += __shfl_xor(pd, 16);   pd += __shfl_xor(pd, 32);
    }
};

// the same of one tile, in fp32 (a lane sees at most 16 of its scores)
struct TileSlope {
    float ds = 0.f, dsd = 0.f, pd = 0.f;
    __device__ __forceinline__ void add(f32x4 p, f32x4 d, f32x4 dist) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ds += d[i];
            dsd = fmaf(d[i], dist[i], dsd);
            pd = fmaf(p[i], dist[i], pd);
        }
    }
    __device__ __forceinline__ void into(Slope &s) const {
        s.ds += ds;
        s.dsd += dsd;
        s.pd += pd;
    }
};

__device__ __forceinline__ float dot_rows(float a0, float a1, float b0, float b1, bool h0, bool h1) {
    return wave_sum((h0 ? a0 * b0 : 0.f) + (h1 ? a1 * b1 : 0.f));
}

// the slow forms: one row or key over its visible partners alone (a masked place's infinity or NaN must not reach it through 0 * inf)
template <typename T> __device__ void dq_slow(const SceneAttnArgs &A, int kvh, const RowState &s, int64_t r, int64_t R) {
    const int lane = threadIdx.x & 63;
    const bool h0 = lane < A.D, h1 = lane + 64 < A.D;
    const int d0 = h0 ? lane : 0, d1 = h1 ? lane + 64 : 0;
    const T *q = reinterpret_cast<const T *>(A.q) + s.row * A.q_rs + s.head * A.q_hs;
    const T *g = reinterpret_cast<const T *>(A.dout) + s.row * A.do_rs + s.head * A.do_hs;
    const T *k = reinterpret_cast<const T *>(A.k) + kvh * A.k_hs, *v = reinterpret_cast<const T *>(A.v) + kvh * A.v_hs;
    const float q0 = to_f(q[d0]), q1 = to_f(q[d1]), g0 = to_f(g[d0]), g1 = to_f(g[d1]);
    const float inv_cap = A.cap > 0.f ? 1.f / A.cap : 0.f, lse = A.lse[kvh * R + r], delta = A.delta[kvh * R + r];
    float a0 = 0.f, a1 = 0.f;
    Slope sl;
    for (int64_t j = s.lo; j < s.hi; ++j) {
        const float k0 = to_f(k[j * A.k_rs + d0]), k1 = to_f(k[j * A.k_rs + d1]);
        const float raw = dot_rows(q0, q1, k0, k1, h0, h1);
        const float dp = dot_rows(g0, g1, to_f(v[j * A.v_rs + d0]), to_f(v[j * A.v_rs + d1]), h0, h1);
        const Grad e = pair_grad(A, raw, dp, inv_cap, s.slope, s.pos, A.kpos + j * A.axes, lse, delta);
        a0 += e.dz * k0;
        a1 += e.dz * k1;
        sl.add(e);
        if (e.dz != e.dz) break;                             // every sum is NaN already
    }
    T *out = reinterpret_cast<T *>(A.dq) + ((int64_t)s.row * A.H + s.head) * A.D;
    if (h0) out[lane] = (T)(a0 * A.scale);
    if (h1) out[lane + 64] = (T)(a1 * A.scale);
    if (A.dsl && lane == 0) A.dsl[kvh * R + r] = sl.row();
}

template <typename T> __device__ void dkv_slow(const SceneAttnArgs &A, int kvh, int64_t key, int64_t R) {
    const int lane = threadIdx.x & 63;
    const bool h0 = lane < A.D, h1 = lane + 64 < A.D;
    const int d0 = h0 ? lane : 0, d1 = h1 ? lane + 64 : 0;
    const T *k = reinterpret_cast<const T *>(A.k) + kvh * A.k_hs + key * A.k_rs, *v = reinterpret_cast<const T *>(A.v) + kvh * A.v_hs + key * A.v_rs;
    const float k0 = to_f(k[d0]), k1 = to_f(k[d1]), v0 = to_f(v[d0]), v1 = to_f(v[d1]);
    const float inv_cap = A.cap > 0.f ? 1.f / A.cap : 0.f;
    float a0 = 0.f, a1 = 0.f, b0 = 0.f, b1 = 0.f;
    const int64_t ra = (int64_t)max(A.key_lo[key], 0) * A.G, rb = (int64_t)min(A.key_hi[key], A.nq) * A.G;
    for (int64_t r = ra; r < rb; ++r) {
        const RowState s = row_state(A, kvh, r, R);
        if (key < s.lo || key >= s.hi) continue;
        const T *q = reinterpret_cast<const T *>(A.q) + s.row * A.q_rs + s.head * A.q_hs;
        const T *g = reinterpret_cast<const T *>(A.dout) + s.row * A.do_rs + s.head * A.do_hs;
        const float q0 = to_f(q[d0]), q1 = to_f(q[d1]), g0 = to_f(g[d0]), g1 = to_f(g[d1]);
        const float raw = dot_rows(q0, q1, k0, k1, h0, h1), dp = dot_rows(g0, g1, v0, v1, h0, h1);
        const Grad e = pair_grad(A, raw, dp, inv_cap, s.slope, s.pos, A.kpos + key * A.axes, A.lse[kvh * R + r], A.delta[kvh * R + r]);
        a0 += e.dz * q0;
        a1 += e.dz * q1;
        b0 += e.p * g0;
        b1 += e.p * g1;
        // every sum is NaN already: nothing that follows changes it (a gradient of NaN, as a loss that overflowed sends back: 4093 causal rows of 96 would be
        // walked for every key, 25 ms for 0.3)
        if (__all((!h0 || (a0 != a0 && b0 != b0)) && (!h1 || (a1 != a1 && b1 != b1)))) break;
    }
    const int64_t at = (key * A.KV + kvh) * A.D;
    T *dk = reinterpret_cast<T *>(A.dk) + at, *dv = reinterpret_cast<T *>(A.dv) + at;
    if (h0) { dk[lane] = (T)(a0 * A.scale); dv[lane] = (T)b0; }
    if (h1) { dk[lane + 64] = (T)(a1 * A.scale); dv[lane + 64] = (T)b1; }
}

// ---------------------------------------------------------------------------------------------------------------------
// dq and dslope: 64 packed rows a workgroup, 16 a wave (columns); K and V tiles in LDS
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DP, int BN, bool CAP, int AX>
__global__ __launch_bounds__(256) void scene_attn_dq_kernel(const SceneAttnArgs A) {
    using X = Tr<T>;
    using L = Tile<T, DP>;
    constexpr int NF = DP / X::KD, DB = DP / 16, PB = X::KB / 16, NC = BN * L::NCH, ROWS = 64;
    static_assert(BN % X::KB == 0, "tile");
    __shared__ u32x4 sk[2][NC], sv[2][NC];
    __shared__ __attribute__((aligned(16))) float sp[2][AX ? AX : 1][BN];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const int kvh = (int)(blockIdx.x % A.KV), both = A.KV * A.key_parts, part = (int)(blockIdx.x / A.KV % A.key_parts);
    const int tiles = gridDim.x / both;
    const int64_t R = (int64_t)A.nq * A.G, r0 = (int64_t)(tiles - 1 - snake(blockIdx.x / both, tiles, max(CUS / both, 1))) * ROWS;
    const Score<CAP, AX, sizeof(T) == 4> S(A);
    const int qa = row_of(r0, A.G), qb = row_of(min(r0 + ROWS, R) - 1, A.G);
    int tlo = uniform(max(A.row_lo[qa], 0)), thi = uniform(min(A.row_hi[qb], A.nk));
    if (A.key_parts > 1) key_part<BN>(tlo, thi, part, A.key_parts);
    const T *K = reinterpret_cast<const T *>(A.k) + kvh * A.k_hs, *V = reinterpret_cast<const T *>(A.v) + kvh * A.v_hs;
    const bool even = A.k_vec == 16 && A.v_vec == 16 && short_rows(A.k_rs, BN, sizeof(T)) && short_rows(A.v_rs, BN, sizeof(T));
    Stage<T, DP, BN, 256> tk, tv;
    tk.offsets([&](int r) { return (uint32_t)(r * A.k_rs * sizeof(T)); }, A.D);
    tv.offsets([&](int r) { return (uint32_t)(r * A.v_rs * sizeof(T)); }, A.D);
    auto issue = [&](int kb, int buf) {
        if (even && kb + BN <= thi) {
            tk.even(sk[buf], K + (int64_t)kb * A.k_rs);
            tv.even(sv[buf], V + (int64_t)kb * A.v_rs);
        } else {
            tk.any(sk[buf], [&](int r) { return K + (int64_t)min(kb + r, thi - 1) * A.k_rs; }, A.D, A.k_vec);
            tv.any(sv[buf], [&](int r) { return V + (int64_t)min(kb + r, thi - 1) * A.v_rs; }, A.D, A.v_vec);
        }
        stage_positions<AX>(sp[buf], A, A.kpos, kb, thi - 1);
    };
    if (tlo < thi) issue(tlo, 0);
    if (tlo + BN < thi) issue(tlo + BN, 1);
    clear_positions<AX>(sp[0], A.axes);
    clear_positions<AX>(sp[1], A.axes);
    const int64_t r = r0 + w * 16 + c;
    const RowState s = row_state(A, kvh, r, R);
    typename X::frag qf[NF], gf[NF];
    const float lse = A.lse[kvh * R + min(r, R - 1)];
    const T *Q = reinterpret_cast<const T *>(A.q) + s.row * A.q_rs + s.head * A.q_hs;
    const T *G = reinterpret_cast<const T *>(A.dout) + s.row * A.do_rs + s.head * A.do_hs;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        qf[f] = as_frag<T>(load_chunk<T>(Q, f * X::KD + g * X::CH, A.D, A.q_vec));
        gf[f] = as_frag<T>(load_chunk<T>(G, f * X::KD + g * X::CH, A.D, A.do_vec));
    }
    const float *o = A.o32 + ((int64_t)s.row * A.H + s.head) * A.D;
    float sum = 0.f;
#pragma unroll
    for (int f = 0; f < NF; ++f) sum = delta_chunk<T>(sum, o, gf[f], f * X::KD + g * X::CH, A.D, A.o32_vec);
    const float delta = group_sum(sum);
    if (part == 0 && g == 0 && r < R) A.delta[kvh * R + r] = delta;
    const int wlo = uniform(__shfl(s.lo, 0)), whi = uniform(__shfl(s.hi, 15));
    const int alo = uniform(__shfl(s.lo, 15)), ahi = uniform(__shfl(s.hi, 0));
    f32x4 acc[DB];
    Slope sl;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};

    int buf = 0;
    for (int kb = tlo; kb < thi; kb += BN, buf ^= 1) {
        landed();
        __syncthreads();
        if (kb > tlo && kb + BN < thi) issue(kb + BN, buf ^ 1);
        TileSlope ts;
#pragma unroll
        for (int j = 0; j < BN / X::KB; ++j) {
            const int k0 = kb + j * X::KB, at = j * X::KB;
            if (k0 >= whi || k0 + X::KB <= wlo) continue;
            f32x4 x[PB], e[PB];
#pragma unroll
            for (int n = 0; n < PB; ++n) {
                x[n] = e[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    const typename X::frag ka = frag_rows<T, DP>(sk[buf], at + n * 16, f, lane);
                    const typename X::frag va = frag_rows<T, DP>(sv[buf], at + n * 16, f, lane);
                    x[n] = mma(ka, qf[f], x[n]);
                    e[n] = mma(va, gf[f], e[n]);
                }
            }
            S.template apply<PB>(x);
#pragma unroll
            for (int n = 0; n < PB; ++n) {
                f32x4 px = {}, py = {}, pz = {};
                if constexpr (AX > 0) read_positions<AX>(sp[buf], at + n * 16 + 4 * g, px, py, pz);
                f32x4 p, ds, dist, t = x[n];
                p = t - lse;
                if constexpr (AX > 0) {
                    dist = S.dist4(s.pos, px, py, pz);
                    p -= s.slope * dist;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[i] = exp2_(p[i]);
                    ds[i] = e[n][i] - delta;
                }
                if (k0 + n * 16 < alo || k0 + n * 16 + 16 > ahi) {       // a masked place is 0, not 0 * inf
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = k0 + n * 16 + 4 * g + i;
                        const bool seen = key >= s.lo && key < s.hi;
                        p[i] = seen ? p[i] : 0.f;
                        ds[i] = seen ? ds[i] : 0.f;
                        if constexpr (CAP) t[i] = seen ? t[i] : 0.f;
                    }
                }
                ds *= p;
                if constexpr (AX > 0)
                    if (A.dsl) ts.add(p, ds, dist);
                e[n] = CAP ? ds * S.slope_of(t) : ds;
            }
            const typename X::frag z = pack_p(e, T());
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const typename X::frag a = frag_cols<DP>(sk[buf], at, d, lane, T());
                acc[d] = mma(a, z, acc[d]);
            }
        }
        if constexpr (AX > 0)
            if (A.dsl) {
                ts.into(sl);
            }
    }
    const int64_t item = (int64_t)s.row * A.H + s.head;
    if constexpr (AX > 0) sl.over_groups();
    if (A.key_parts > 1) {
        if (r < R) {
#pragma unroll
            for (int d = 0; d < DB; ++d) store4(A.part + (item * A.key_parts + part) * A.D, acc[d] * A.scale, d * 16 + g * 4, A.D, A.D % 4 == 0);
            if (AX > 0 && g == 0) {
                double *st = reinterpret_cast<double *>(A.stat) + (item * A.key_parts + part) * 3;
                st[0] = sl.ds; st[1] = sl.dsd; st[2] = sl.pd;
            }
        }
        return;
    }
    const float dslope = AX > 0 ? sl.row() : 0.f;
    bool fine = finite_(dslope);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[d][i] *= A.scale;
            fine = fine && finite_(acc[d][i]);
        }
    if (r < R) {
        T *out = reinterpret_cast<T *>(A.dq) + item * A.D;
#pragma unroll
        for (int d = 0; d < DB; ++d) store4(out, acc[d], d * 16 + g * 4, A.D, A.o_vec != 0);
        if (AX > 0 && A.dsl && g == 0) A.dsl[kvh * R + r] = dslope;
    }
    uint64_t bad = __ballot(!fine && r < R);
    while (bad) {
        const int src = __builtin_ctzll(bad) & 15;
        bad &= ~(0x0001000100010001ull << src);
        const int64_t rr = r - c + src;
        dq_slow<T>(A, kvh, row_state(A, kvh, rr, R), rr, R);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// dk and dv: 64 keys a workgroup, 16 a wave (columns); tiles of BM packed rows (q, do and what belongs to a row) in LDS.
// parts > 1: a workgroup takes one part of the rows that see its keys and leaves fp32 sums; scene_attn_dkv_join_kernel adds them.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DP, int BM, bool CAP, int AX>
__global__ __launch_bounds__(256, DP <= 32 ? 4 : DP <= 96 ? 3 : 2) void scene_attn_dkv_kernel(const SceneAttnArgs A) {
    using X = Tr<T>;
    using L = Tile<T, DP>;
    constexpr int NF = DP / X::KD, DB = DP / 16, PB = X::KB / 16, NC = BM * L::NCH, KEYS = 64, NV = 5 + AX;
    static_assert(BM % X::KB == 0 && BM <= 64, "tile");
    __shared__ u32x4 sq[2][NC], sg[2][NC];
    __shared__ __attribute__((aligned(16))) float srow[2][NV][BM];      // lse, delta, lo, hi, slope, position
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const int kvh = (int)(blockIdx.x % A.KV), part = (int)(blockIdx.x / A.KV % A.parts);
    const int64_t R = (int64_t)A.nq * A.G;
    const int both = A.KV * A.parts, k0 = (int)snake(blockIdx.x / both, gridDim.x / both, max(CUS / both, 1)) * KEYS, kw = k0 + w * 16;
    const Score<CAP, AX, sizeof(T) == 4> S(A);
    // the packed rows that see the workgroup's keys (this part of them)
    int64_t ra = (int64_t)max(A.key_lo[k0], 0) * A.G, rb = (int64_t)min(A.key_hi[min(k0 + KEYS - 1, A.nk - 1)], A.nq) * A.G;
    if (A.parts > 1) {
        const int64_t n = max(rb - ra, (int64_t)0) + A.parts - 1, per = ((n <= 0xffffffffll ? (int64_t)((uint32_t)n / (uint32_t)A.parts) : n / A.parts) + BM - 1) / BM * BM;
        ra += per * part;
        rb = min(rb, ra + per);
    }
    // packed rows start at a row's first head and BM holds whole rows
    const bool even = BM % A.G == 0 && A.q_vec == 16 && A.do_vec == 16 && short_rows(A.q_rs, BM, sizeof(T)) && short_rows(A.do_rs, BM, sizeof(T)) &&
                      short_rows(A.q_hs, BM, sizeof(T)) && short_rows(A.do_hs, BM, sizeof(T));
    Stage<T, DP, BM, 256> tq, tg;
    tq.offsets([&](int r) { return (uint32_t)((r / A.G * A.q_rs + r % A.G * A.q_hs) * sizeof(T)); }, A.D);
    tg.offsets([&](int r) { return (uint32_t)((r / A.G * A.do_rs + r % A.G * A.do_hs) * sizeof(T)); }, A.D);
    auto issue = [&](int64_t rbase, int buf) {              // rows behind the last one: the last one again, masked below
        auto at = [&](int r, int64_t rs, int64_t hs) {
            const int64_t rr = min(rbase + r, rb - 1), row = row_of(rr, A.G);
            return row * rs + (kvh * A.G + (rr - row * A.G)) * hs;
        };
        const T *Q = reinterpret_cast<const T *>(A.q), *G = reinterpret_cast<const T *>(A.dout);
        if (even && rbase + BM <= rb) {
            tq.even(sq[buf], Q + at(0, A.q_rs, A.q_hs));
            tg.even(sg[buf], G + at(0, A.do_rs, A.do_hs));
        } else {
            tq.any(sq[buf], [&](int r) { return Q + at(r, A.q_rs, A.q_hs); }, A.D, A.q_vec);
            tg.any(sg[buf], [&](int r) { return G + at(r, A.do_rs, A.do_hs); }, A.D, A.do_vec);
        }
        const int64_t rr = min(rbase + lane, rb - 1), row = row_of(rr, A.G);
        if (w == 0) {
            stage_values<BM>(srow[buf][0], A.lse + kvh * R + rr);
            stage_values<BM>(srow[buf][1], A.delta + kvh * R + rr);
        } else if (w == 1) {
            stage_values<BM>(srow[buf][2], A.row_lo + row);
            stage_values<BM>(srow[buf][3], A.row_hi + row);
        } else if (AX > 0 && w == 2) {
            stage_values<BM>(srow[buf][4], A.slopes + kvh * A.G + (rr - row * A.G));
            stage_values<BM>(srow[buf][5], A.qpos + row * A.axes);
        } else if (AX > 1) {
            stage_values<BM>(srow[buf][6], A.qpos + row * A.axes + 1);
            if (A.axes > 2) stage_values<BM>(srow[buf][NV - 1], A.qpos + row * A.axes + 2);
        }
    };
    if (ra < rb) issue(ra, 0);
    if (ra + BM < rb) issue(ra + BM, 1);
    if (AX > 1 && A.axes < 3)
        for (int i = tid; i < 2 * BM; i += 256) srow[i / BM][NV - 1][i % BM] = 0.f;

    typename X::frag kf[NF], vf[NF];
    float kpos[3];
    const int kk = min(kw + c, A.nk - 1);
    const T *K = reinterpret_cast<const T *>(A.k) + (int64_t)kk * A.k_rs + kvh * A.k_hs, *V = reinterpret_cast<const T *>(A.v) + (int64_t)kk * A.v_rs + kvh * A.v_hs;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        kf[f] = as_frag<T>(load_chunk<T>(K, f * X::KD + g * X::CH, A.D, A.k_vec));
        vf[f] = as_frag<T>(load_chunk<T>(V, f * X::KD + g * X::CH, A.D, A.v_vec));
    }
#pragma unroll
    for (int a = 0; a < 3; ++a) kpos[a] = a < AX && a < A.axes ? A.kpos[(int64_t)kk * A.axes + a] : 0.f;
    // the rows that see a key of this wave
    const int64_t wa = (int64_t)max(A.key_lo[min(kw, A.nk - 1)], 0) * A.G, wb = (int64_t)min(A.key_hi[min(kw + 15, A.nk - 1)], A.nq) * A.G;
    f32x4 dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[d] = dv[d] = f32x4{0.f, 0.f, 0.f, 0.f};

    int buf = 0;
    for (int64_t rbase = ra; rbase < rb; rbase += BM, buf ^= 1) {
        landed();
        __syncthreads();
        if (rbase > ra && rbase + BM < rb) issue(rbase + BM, buf ^ 1);
#pragma unroll
        for (int j = 0; j < BM / X::KB; ++j) {
            const int64_t r0 = rbase + j * X::KB;
            const int at = j * X::KB;
            if (r0 >= wb || r0 + X::KB <= wa || r0 >= rb) continue;
            // bounds never decrease: the last row has the latest lo, the first the earliest hi
            const int lo_last = uniform(__float_as_int(srow[buf][2][at + X::KB - 1])), hi_first = uniform(__float_as_int(srow[buf][3][at]));
            const bool masked = kw < lo_last || kw + 16 > hi_first || r0 + X::KB > rb;
            f32x4 p[PB], z[PB];
#pragma unroll
            for (int n = 0; n < PB; ++n) {
                p[n] = z[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    const typename X::frag qa = frag_rows<T, DP>(sq[buf], at + n * 16, f, lane);
                    const typename X::frag ga = frag_rows<T, DP>(sg[buf], at + n * 16, f, lane);
                    p[n] = mma(qa, kf[f], p[n]);
                    z[n] = mma(ga, vf[f], z[n]);
                }
            }
            S.template apply<PB>(p);
#pragma unroll
            for (int n = 0; n < PB; ++n) {
                auto col = [&](int v) { return *reinterpret_cast<const f32x4 *>(&srow[buf][v][at + n * 16 + 4 * g]); };
                const f32x4 lse = col(0), delta = col(1);
                f32x4 slope = {}, px = {}, py = {}, pz = {};
                if constexpr (AX > 0) {
                    slope = col(4) * LOG2E;
                    px = col(5);
                }
                if constexpr (AX > 1) {
                    py = col(6);
                    pz = col(NV - 1);
                }
                f32x4 t = p[n];
                p[n] = t - lse;
                if constexpr (AX > 0) p[n] -= slope * S.dist4(kpos, px, py, pz);
                z[n] -= delta;
#pragma unroll
                for (int i = 0; i < 4; ++i) p[n][i] = exp2_(p[n][i]);
                if (masked) {                           // a masked place is 0, not 0 * inf
                    const f32x4 lo = col(2), hi = col(3);
                    const int key = kw + c;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool seen = key >= __float_as_int(lo[i]) && key < __float_as_int(hi[i]) && r0 + n * 16 + 4 * g + i < rb;
                        p[n][i] = seen ? p[n][i] : 0.f;
                        z[n][i] = seen ? z[n][i] : 0.f;
                        if constexpr (CAP) t[i] = seen ? t[i] : 0.f;
                    }
                }
                z[n] *= p[n];
                if constexpr (CAP) z[n] *= S.slope_of(t);
            }
            const typename X::frag pf = pack_p(p, T()), zf = pack_p(z, T());
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const typename X::frag ga = frag_cols<DP>(sg[buf], at, d, lane, T());
                const typename X::frag qa = frag_cols<DP>(sq[buf], at, d, lane, T());
                dv[d] = mma(ga, pf, dv[d]);
                dk[d] = mma(qa, zf, dk[d]);
            }
        }
    }
    const int key = kw + c;
    const int64_t at = ((int64_t)key * A.KV + kvh) * A.D;
    bool fine = true;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            dk[d][i] *= A.scale;
            fine = fine && finite_(dk[d][i]) && finite_(dv[d][i]);
        }
    if (A.parts > 1) {
        const int64_t n = (int64_t)A.nk * A.KV * A.D;
        if (key < A.nk) {
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                store4(A.part2 + 2 * part * n + at, dk[d], d * 16 + g * 4, A.D, A.D % 4 == 0);
                store4(A.part2 + (2 * part + 1) * n + at, dv[d], d * 16 + g * 4, A.D, A.D % 4 == 0);
            }
        }
        return;
    }
    if (key < A.nk) {
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            store4(reinterpret_cast<T *>(A.dk) + at, dk[d], d * 16 + g * 4, A.D, A.o_vec != 0);
            store4(reinterpret_cast<T *>(A.dv) + at, dv[d], d * 16 + g * 4, A.D, A.o_vec != 0);
        }
    }
    uint64_t bad = __ballot(!fine && key < A.nk);
    while (bad) {
        const int src = __builtin_ctzll(bad) & 15;
        bad &= ~(0x0001000100010001ull << src);
        dkv_slow<T>(A, kvh, key - c + src, R);
    }
}

// dq (and a row's part of dslope) from the parts' sums, in order; 32 lanes per (row, head), four columns a lane
template <typename T> __global__ __launch_bounds__(256) void scene_attn_dq_join_kernel(const SceneAttnArgs A) {
    const int lane = threadIdx.x & 63, P = A.key_parts, d = (lane & 31) * 4, vec = A.D % 4 == 0 ? 16 : 4;
    const int64_t items = (int64_t)A.nq * A.H, R = (int64_t)A.nq * A.G, own = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), item = min(own, items - 1);
    const int64_t row = item / A.H;
    const int head = (int)(item - row * A.H), kvh = head / A.G;
    const int64_t r = row * A.G + head - kvh * A.G;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < P; ++i) a += __builtin_bit_cast(f32x4, load_chunk<float>(A.part + (item * P + i) * A.D, d, A.D, vec));
    Slope s;
    if (A.dsl)
        for (int i = 0; i < P; ++i) {
            const double *st = reinterpret_cast<const double *>(A.stat) + (item * P + i) * 3;
            s.ds += st[0];
            s.dsd += st[1];
            s.pd += st[2];
        }
    if (own < items) {
        store4(reinterpret_cast<T *>(A.dq) + item * A.D, a, d, A.D, A.o_vec != 0);
        if (A.dsl && d == 0) A.dsl[kvh * R + r] = s.row();
    }
    const bool fine = own >= items || (finite_(s.row()) && finite_(a[0]) && finite_(a[1]) && finite_(a[2]) && finite_(a[3]));
    const uint64_t bad = __ballot(!fine);
    for (int h = 0; h < 2; ++h)                              // the wave's two pairs
        if (bad >> (32 * h) & 0xffffffffull) dq_slow<T>(A, __shfl(kvh, 32 * h), row_state(A, __shfl(kvh, 32 * h), __shfl(r, 32 * h), R), __shfl(r, 32 * h), R);
}

// dk and dv from the parts' sums, in order; 32 lanes per (key, kv head), four columns a lane
template <typename T> __global__ __launch_bounds__(256) void scene_attn_dkv_join_kernel(const SceneAttnArgs A) {
    const int lane = threadIdx.x & 63, d = (lane & 31) * 4, vec = A.D % 4 == 0 ? 16 : 4;
    const int64_t items = (int64_t)A.nk * A.KV, n = items * A.D, own = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), item = min(own, items - 1);
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < A.parts; ++i) {
        a += __builtin_bit_cast(f32x4, load_chunk<float>(A.part2 + 2 * i * n + item * A.D, d, A.D, vec));
        b += __builtin_bit_cast(f32x4, load_chunk<float>(A.part2 + (2 * i + 1) * n + item * A.D, d, A.D, vec));
    }
    bool fine = true;
    if (own < items) {
        store4(reinterpret_cast<T *>(A.dk) + item * A.D, a, d, A.D, A.o_vec != 0);
        store4(reinterpret_cast<T *>(A.dv) + item * A.D, b, d, A.D, A.o_vec != 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) fine = fine && finite_(a[i]) && finite_(b[i]);
    }
    const uint64_t bad = __ballot(!fine);
    for (int h = 0; h < 2; ++h)                              // the wave's two pairs
        if (bad >> (32 * h) & 0xffffffffull) {
            const int64_t it = __shfl(item, 32 * h);
            dkv_slow<T>(A, (int)(it % A.KV), it / A.KV, (int64_t)A.nq * A.G);
        }
}

template <typename T, int DP, int BN, bool CAP, int AX> hipError_t launch_bwd(const SceneAttnArgs &A, hipStream_t st) {
    const int64_t tiles = ((int64_t)A.nq * A.G + 63) / 64;
    if (tiles > 0 && A.dq) hipLaunchKernelGGL((scene_attn_dq_kernel<T, DP, BN, CAP, AX>), dim3((unsigned)(tiles * A.KV * A.key_parts)), dim3(256), 0, st, A);
    if (tiles > 0 && A.dq && A.key_parts > 1) hipLaunchKernelGGL((scene_attn_dq_join_kernel<T>), dim3((unsigned)(((int64_t)A.nq * A.H + 7) / 8)), dim3(256), 0, st, A);
    if (A.nk > 0 && A.dk) {
        hipLaunchKernelGGL((scene_attn_dkv_kernel<T, DP, BN, CAP, AX>), dim3((unsigned)(((int64_t)A.nk + 63) / 64 * A.KV * A.parts)), dim3(256), 0, st, A);
        if (A.parts > 1) hipLaunchKernelGGL((scene_attn_dkv_join_kernel<T>), dim3((unsigned)(((int64_t)A.nk * A.KV + 7) / 8)), dim3(256), 0, st, A);
    }
    return hipGetLastError();
}
template <typename T, int DP, int BN> hipError_t pick_bwd(const SceneAttnArgs &A, hipStream_t st) {
    if (A.cap > 0.f) return A.axes == 0 ? launch_bwd<T, DP, BN, true, 0>(A, st) : A.axes == 1 ? launch_bwd<T, DP, BN, true, 1>(A, st) : launch_bwd<T, DP, BN, true, 3>(A, st);
    return A.axes == 0 ? launch_bwd<T, DP, BN, false, 0>(A, st) : A.axes == 1 ? launch_bwd<T, DP, BN, false, 1>(A, st) : launch_bwd<T, DP, BN, false, 3>(A, st);
}
template <typename T> hipError_t run_bwd(const SceneAttnArgs &A, float *dslopes, hipStream_t st) {
    const int64_t n = (int64_t)A.nq * A.H;
    if (n > 0 && !A.dq) hipLaunchKernelGGL((scene_attn_delta_kernel<T>), dim3((unsigned)((n + 63) / 64)), dim3(256), 0, st, A);
    const int D = A.D;
    hipError_t e;
    if constexpr (sizeof(T) == 2) e = D <= 32 ? pick_bwd<T, 32, 64>(A, st) : D <= 64 ? pick_bwd<T, 64, 64>(A, st) : D <= 96 ? pick_bwd<T, 96, 32>(A, st) : pick_bwd<T, 128, 32>(A, st);
    else e = D <= 16 ? pick_bwd<T, 16, 64>(A, st) : D <= 32 ? pick_bwd<T, 32, 32>(A, st) : D <= 48 ? pick_bwd<T, 48, 32>(A, st) : D <= 64 ? pick_bwd<T, 64, 32>(A, st)
           : D <= 96 ? pick_bwd<T, 96, 32>(A, st) : pick_bwd<T, 128, 32>(A, st);
    if (e != hipSuccess) return e;
    if (dslopes) hipLaunchKernelGGL(scene_attn_dslope_kernel, dim3(A.H), dim3(1024), 0, st, A.nq, A.G, A.dsl, dslopes);
    return hipGetLastError();
}

}  // namespace sattn

// one object file per type (the Makefile compiles this source twice)
#ifdef SCENE_ATTN_BF16
extern "C" hipError_t dn_scene_attn_bwd_bf16(const SceneAttnArgs *A, float *dslopes, hipStream_t st) { return sattn::run_bwd<sattn::bf16>(*A, dslopes, st); }
#else
extern "C" hipError_t dn_scene_attn_bwd_f32(const SceneAttnArgs *A, float *dslopes, hipStream_t st) { return sattn::run_bwd<float>(*A, dslopes, st); }
// Parts of the rows in the dk / dv kernel.  seen: rows that see a key, where most do (the longest tile is what the rest waits for); 64 keys see about 64 more.
// - As many as give the chip nine workgroups a CU (places for two or three at once: unlike tiles level out, and no round is left half empty), beyond 8 parts only
//   what gives four: the join reads two fp32 sums a part.  bf16, 8 heads to 2, dk and dv with four and with nine: 16384 causal rows of 96, 1499 us and
//   1218, of 64 960 and 781, all seen 2927 and 2391; 24000 causal, 4423 and 2646; 4093 causal (8 and 16 parts), 112 + 10 to join and 110 + 16.
// - None below 128 packed rows of those.  fp32, 2400 causal rows in two scenes, one head of 100: the whole backward and forward 151 us with at least 256, 126 with
//   128; 1000 rows, 4 heads of 72 to one, backward alone: 199 us with 512, 134 with 256, 122 with 128.  48 scenes of 60 - 340 rows, 4 heads of 32 to 2: 52 + 7
//   to join with 256, 53 + 10 with 128: there the chip is full already.
extern "C" int dn_scene_attn_bwd_parts(int64_t nk, int KV, int G, int64_t seen) {
    const int64_t groups = (nk + 63) / 64 * KV;
    if (!groups) return 1;
    const int64_t four = 1024 / groups, nine = 2304 / groups, most = (seen + 64) * G / 128;
    int64_t parts = four > 8 ? four : nine < 8 ? nine : 8;
    parts = parts < most ? parts : most;
    return (int)(parts < 1 ? 1 : parts < 16 ? parts : 16);
}
#endif
