// Backward of the scene attention (scene_attn.h has the mathematics and the layout).
//     p_ij = 2^(x_ij - lse_i),  dp_ij = do_i.v_j,  ds_ij = p_ij (dp_ij - delta_i),  delta_i = do_i.o_i
//     dslope_h = - sum_ij ds_ij |pos_i - pos_j|;   dz_ij = ds_ij (1 - tanh^2) scale;   dq_i = sum_j dz_ij k_j,  dk_j = sum_i dz_ij q_i,
//     dv_j = sum_i p_ij do_i
// Two kernels recompute p from the saved lse, one with query rows on the lanes' columns (dq, dslope), one with keys on them (dk, dv): every
// sum has one owner and one order, so results repeat bit for bit.
// delta is taken from the unrounded output.  What is left of its error (in bf16 the forward's p was rounded for its second product) moves
// every ds of a row by p_ij e_i.  dslope, a sum over all scores of which most cancels, does not forgive that, but a row's ds have to
// add up to nothing, so e_i = - sum_j ds_ij is known and what it did to dslope is taken back: three sums per row instead of one.
#include "scene_attn.h"

namespace sattn {

// delta[kvh][row G + g] = sum_d do * o; a wave takes 16 (row, head) pairs, four lanes each
template <typename T> __global__ __launch_bounds__(256) void scene_attn_delta_kernel(const SceneAttnArgs A) {
    const int64_t n = (int64_t)A.nq * A.H, i = (int64_t)blockIdx.x * 64 + (threadIdx.x >> 2);
    const int part = threadIdx.x & 3;
    float s = 0.f;
    if (i < n) {
        const int64_t row = i / A.H;
        const int head = (int)(i - row * A.H);
        const T *g = reinterpret_cast<const T *>(A.dout) + row * A.do_rs + head * A.do_hs;
        const float *o = A.o32 + i * A.D;
        for (int d = part; d < A.D; d += 4) s += to_f(g[d]) * o[d];
    }
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    if (i < n && part == 0) {
        const int64_t row = i / A.H;
        const int head = (int)(i - row * A.H), kvh = head / A.G;
        A.delta[(int64_t)kvh * A.nq * A.G + row * A.G + (head - kvh * A.G)] = s;
    }
}

// dslopes[h] = sum over the rows of what the dq kernel left per packed row; one workgroup per head, fp64, fixed order
__global__ __launch_bounds__(256) void scene_attn_dslope_kernel(int nq, int G, const float *__restrict__ part, float *__restrict__ out) {
    __shared__ double sh[256];
    const int h = blockIdx.x, kvh = h / G, g = h - kvh * G;
    const float *p = part + (int64_t)kvh * nq * G + g;
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < nq; i += 256) s += p[i * G];
    sh[threadIdx.x] = s;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[h] = (float)sh[0];
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
    float ds = 0.f, dsd = 0.f, pd = 0.f;
    __device__ __forceinline__ void add(const Grad &g, bool seen) {
        const float d = seen ? g.ds : 0.f, p = seen ? g.p : 0.f;
        ds += d;
        dsd += d * g.dist;
        pd += p * g.dist;
    }
    __device__ __forceinline__ float row() const { return ds * pd - dsd; }
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
        sl.add(e, true);
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
    }
    const int64_t at = (key * A.KV + kvh) * A.D;
    T *dk = reinterpret_cast<T *>(A.dk) + at, *dv = reinterpret_cast<T *>(A.dv) + at;
    if (h0) { dk[lane] = (T)(a0 * A.scale); dv[lane] = (T)b0; }
    if (h1) { dk[lane + 64] = (T)(a1 * A.scale); dv[lane + 64] = (T)b1; }
}

// ---------------------------------------------------------------------------------------------------------------------
// dq and dslope: 64 packed rows a workgroup, 16 a wave (columns); K and V tiles in LDS
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DP, int BN>
__global__ __launch_bounds__(256) void scene_attn_dq_kernel(const SceneAttnArgs A) {
    using X = Tr<T>;
    using L = Tile<T, DP>;
    constexpr int NF = DP / X::KD, DB = DP / 16, PB = X::KB / 16, NC = BN * L::NCH, PER = NC / 256;
    static_assert(NC % 256 == 0 && BN % X::KB == 0, "tile");
    __shared__ u32x4 sk[NC], sv[NC];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const int kvh = (int)(blockIdx.x % A.KV);
    const int64_t R = (int64_t)A.nq * A.G, r0 = (int64_t)(gridDim.x / A.KV - 1 - blockIdx.x / A.KV) * 64, r = r0 + w * 16 + c;
    const RowState s = row_state(A, kvh, r, R);
    const float lse = A.lse[kvh * R + min(r, R - 1)], delta = A.delta[kvh * R + min(r, R - 1)];
    const T *Q = reinterpret_cast<const T *>(A.q) + s.row * A.q_rs + s.head * A.q_hs;
    const T *G = reinterpret_cast<const T *>(A.dout) + s.row * A.do_rs + s.head * A.do_hs;
    typename X::frag qf[NF], gf[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        qf[f] = as_frag<T>(load_chunk<T>(Q, f * X::KD + g * X::CH, A.D, A.q_vec));
        gf[f] = as_frag<T>(load_chunk<T>(G, f * X::KD + g * X::CH, A.D, A.do_vec));
    }
    const int qa = (int)(r0 / A.G), qb = (int)((min(r0 + 64, R) - 1) / A.G);
    const int tlo = max(A.row_lo[qa], 0), thi = min(A.row_hi[qb], A.nk);
    const int wlo = __builtin_amdgcn_readfirstlane(__shfl(s.lo, 0)), whi = __builtin_amdgcn_readfirstlane(__shfl(s.hi, 15));
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
    f32x4 acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    Slope sl;
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
#pragma unroll
        for (int j = 0; j < BN / X::KB; ++j) {
            const int k0 = kb + j * X::KB;
            if (k0 >= whi || k0 + X::KB <= wlo) continue;
            f32x4 dz[PB];
#pragma unroll
            for (int b = 0; b < PB; ++b) {
                f32x4 a = {0.f, 0.f, 0.f, 0.f}, e = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    a = mma(frag_rows<T, DP>(sk, j * X::KB + b * 16, f, lane), qf[f], a);
                    e = mma(frag_rows<T, DP>(sv, j * X::KB + b * 16, f, lane), gf[f], e);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = k0 + b * 16 + 4 * g + i;
                    const bool seen = key >= s.lo && key < s.hi;
                    const Grad q = pair_grad(A, a[i], e[i], inv_cap, s.slope, s.pos, A.kpos + (int64_t)min(key, A.nk - 1) * A.axes, lse, delta);
                    dz[b][i] = seen ? q.dz : 0.f;
                    if (A.dsl) sl.add(q, seen);
                }
            }
            const typename X::frag p = pack_p(dz, T());
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[d] = mma(frag_cols<DP>(sk, j * X::KB, d, lane, T()), p, acc[d]);
        }
    }
    sl.ds = group_sum(sl.ds);
    sl.dsd = group_sum(sl.dsd);
    sl.pd = group_sum(sl.pd);
    const float dslope = sl.row();
    bool fine = finite_(dslope);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[d][i] *= A.scale;
            fine = fine && finite_(acc[d][i]);
        }
    if (r < R) {
        T *out = reinterpret_cast<T *>(A.dq) + ((int64_t)s.row * A.H + s.head) * A.D;
#pragma unroll
        for (int d = 0; d < DB; ++d) store4(out, acc[d], d * 16 + g * 4, A.D, A.o_vec != 0);
        if (A.dsl && g == 0) A.dsl[kvh * R + r] = dslope;
    }
    uint64_t bad = __ballot(!fine && r < R);
    while (bad) {
        const int src = __builtin_ctzll(bad) & 15;
        bad &= ~(0x0001000100010001ull << src);
        const RowState t = row_state(A, kvh, r0 + w * 16 + src, R);
        dq_slow<T>(A, kvh, t, r0 + w * 16 + src, R);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// dk and dv: 64 keys a workgroup, 16 a wave (columns); tiles of BM packed rows (q, do and what belongs to a row) in LDS
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DP, int BM>
__global__ __launch_bounds__(256) void scene_attn_dkv_kernel(const SceneAttnArgs A) {
    using X = Tr<T>;
    using L = Tile<T, DP>;
    constexpr int NF = DP / X::KD, DB = DP / 16, PB = X::KB / 16, NC = BM * L::NCH, PER = NC / 256;
    static_assert(NC % 256 == 0 && BM % X::KB == 0 && BM <= 64, "tile");
    __shared__ u32x4 sq[NC], sg[NC];
    __shared__ float srow[BM][8];                // lse, delta, slope, lo, hi, position
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const int kvh = (int)(blockIdx.x % A.KV);
    const int64_t R = (int64_t)A.nq * A.G;
    const int k0 = (int)(blockIdx.x / A.KV) * 64, key = k0 + w * 16 + c, kk = min(key, A.nk - 1);
    const T *K = reinterpret_cast<const T *>(A.k) + (int64_t)kk * A.k_rs + kvh * A.k_hs, *V = reinterpret_cast<const T *>(A.v) + (int64_t)kk * A.v_rs + kvh * A.v_hs;
    typename X::frag kf[NF], vf[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        kf[f] = as_frag<T>(load_chunk<T>(K, f * X::KD + g * X::CH, A.D, A.k_vec));
        vf[f] = as_frag<T>(load_chunk<T>(V, f * X::KD + g * X::CH, A.D, A.v_vec));
    }
    float kpos[3] = {0.f, 0.f, 0.f};
    for (int a = 0; a < A.axes; ++a) kpos[a] = A.kpos[(int64_t)kk * A.axes + a];
    const int64_t ra = (int64_t)max(A.key_lo[k0], 0) * A.G, rb = (int64_t)min(A.key_hi[min(k0 + 63, A.nk - 1)], A.nq) * A.G;
    const int64_t wa = (int64_t)max(A.key_lo[min(k0 + w * 16, A.nk - 1)], 0) * A.G;
    const int64_t wb = (int64_t)min(A.key_hi[min(k0 + w * 16 + 15, A.nk - 1)], A.nq) * A.G;
    const float inv_cap = A.cap > 0.f ? 1.f / A.cap : 0.f;

    u32x4 rq[PER], rg[PER];
    float extra[8];
    auto fetch = [&](int64_t rbase) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = tid + i * 256, ch = e % L::NCH;
            const int64_t rr = rbase + e / L::NCH;
            const u32x4 z = {0u, 0u, 0u, 0u};
            rq[i] = rg[i] = z;
            if (rr < rb) {
                const int64_t row = rr / A.G, head = kvh * A.G + (rr - row * A.G);
                rq[i] = load_chunk<T>(reinterpret_cast<const T *>(A.q) + row * A.q_rs + head * A.q_hs, ch * X::CH, A.D, A.q_vec);
                rg[i] = load_chunk<T>(reinterpret_cast<const T *>(A.dout) + row * A.do_rs + head * A.do_hs, ch * X::CH, A.D, A.do_vec);
            }
        }
        if (tid < BM) {
            const int64_t rr = rbase + tid;
            const RowState s = row_state(A, kvh, rr, R);
            const bool in = rr < rb;
            extra[0] = in ? A.lse[kvh * R + rr] : 0.f;
            extra[1] = in ? A.delta[kvh * R + rr] : 0.f;
            extra[2] = s.slope;
            extra[3] = __int_as_float(in ? s.lo : 0);
            extra[4] = __int_as_float(in ? s.hi : 0);
            extra[5] = s.pos[0]; extra[6] = s.pos[1]; extra[7] = s.pos[2];
        }
    };
    f32x4 dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[d] = dv[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (ra < rb) fetch(ra);
    for (int64_t rbase = ra; rbase < rb; rbase += BM) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = tid + i * 256;
            sq[L::slot(e / L::NCH, e % L::NCH)] = rq[i];
            sg[L::slot(e / L::NCH, e % L::NCH)] = rg[i];
        }
        if (tid < BM) {
#pragma unroll
            for (int i = 0; i < 8; ++i) srow[tid][i] = extra[i];
        }
        __syncthreads();
        if (rbase + BM < rb) fetch(rbase + BM);
#pragma unroll
        for (int j = 0; j < BM / X::KB; ++j) {
            const int64_t r0 = rbase + j * X::KB;
            if (r0 >= wb || r0 + X::KB <= wa) continue;
            f32x4 p[PB], dz[PB];
#pragma unroll
            for (int b = 0; b < PB; ++b) {
                f32x4 a = {0.f, 0.f, 0.f, 0.f}, e = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    a = mma(frag_rows<T, DP>(sq, j * X::KB + b * 16, f, lane), kf[f], a);
                    e = mma(frag_rows<T, DP>(sg, j * X::KB + b * 16, f, lane), vf[f], e);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float *s = srow[j * X::KB + b * 16 + 4 * g + i];
                    const bool seen = key >= __float_as_int(s[3]) && key < __float_as_int(s[4]);
                    const Grad q = pair_grad(A, a[i], e[i], inv_cap, s[2], s + 5, kpos, s[0], s[1]);
                    p[b][i] = seen ? q.p : 0.f;
                    dz[b][i] = seen ? q.dz : 0.f;
                }
            }
            const typename X::frag pf = pack_p(p, T()), zf = pack_p(dz, T());
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                dv[d] = mma(frag_cols<DP>(sg, j * X::KB, d, lane, T()), pf, dv[d]);
                dk[d] = mma(frag_cols<DP>(sq, j * X::KB, d, lane, T()), zf, dk[d]);
            }
        }
    }
    bool fine = true;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            dk[d][i] *= A.scale;
            fine = fine && finite_(dk[d][i]) && finite_(dv[d][i]);
        }
    if (key < A.nk) {
        const int64_t at = ((int64_t)key * A.KV + kvh) * A.D;
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
        dkv_slow<T>(A, kvh, k0 + w * 16 + src, R);
    }
}

template <typename T, int DP, int BN> hipError_t launch_bwd(const SceneAttnArgs &A, float *dslopes, hipStream_t st) {
    const int64_t n = (int64_t)A.nq * A.H, tiles = ((int64_t)A.nq * A.G + 63) / 64;
    if (n > 0) {
        hipLaunchKernelGGL((scene_attn_delta_kernel<T>), dim3((unsigned)((n + 63) / 64)), dim3(256), 0, st, A);
        if (A.dq) hipLaunchKernelGGL((scene_attn_dq_kernel<T, DP, BN>), dim3((unsigned)(tiles * A.KV)), dim3(256), 0, st, A);
    }
    if (A.nk > 0 && A.dk) hipLaunchKernelGGL((scene_attn_dkv_kernel<T, DP, BN>), dim3((unsigned)(((int64_t)A.nk + 63) / 64 * A.KV)), dim3(256), 0, st, A);
    if (dslopes) hipLaunchKernelGGL(scene_attn_dslope_kernel, dim3(A.H), dim3(256), 0, st, A.nq, A.G, A.dsl, dslopes);
    return hipGetLastError();
}

}  // namespace sattn

extern "C" hipError_t dn_scene_attn_bwd(const SceneAttnArgs *A, int bf, float *dslopes, hipStream_t st) {
    using namespace sattn;
    const int D = A->D;
    if (bf) return D <= 32 ? launch_bwd<bf16, 32, 64>(*A, dslopes, st) : D <= 64 ? launch_bwd<bf16, 64, 64>(*A, dslopes, st) : launch_bwd<bf16, 128, 32>(*A, dslopes, st);
    return D <= 16 ? launch_bwd<float, 16, 64>(*A, dslopes, st) : D <= 32 ? launch_bwd<float, 32, 64>(*A, dslopes, st)
         : D <= 64 ? launch_bwd<float, 64, 32>(*A, dslopes, st) : launch_bwd<float, 128, 32>(*A, dslopes, st);
}
