// Forward of the scene attention (scene_attn.h has the mathematics and the layout).
//
// One workgroup: 64 packed rows of one kv head, 16 per wave (or 128, 32 per wave); K and V tiles of BN keys in LDS twice over, the next
// tile's loads going straight into the other copy while the current one is worked on.  A wave skips 16-key blocks that none of its rows sees, so a tile that holds
// several small scenes costs each wave its own scenes only.
//
// Bound by vector instructions, by counters (masked places and filled-up tiles among them): bf16 with cap, three axes and the exact second product 40 a
// visible score (32 scenes of 500 rows; issuing in 72 % of the CUs' busy clocks), with cap and one axis 22 (long causal rows of 128; 75 %), without either and with
// the exact product 15 (4093 causal rows of 96; 59 %, LDS reads 45 %).  Three of them run at a quarter of the rate: exponential, quotient, root.
// Measured, bf16, all keys seen: 16384 rows of 8 heads of 96 to 2, 0.87 ms (945 TFLOP/s, a plain 8192^3 product reaches 1195); capped 1.44 ms; 128 wide 1.08 ms
// (1015 TFLOP/s).  Small scenes are bound by one workgroup's chain of loads: 4096 fp32 scenes of ten rows, 4 heads of 16, 25 us (42 MB, 1.7 TB/s); four times
// the workgroups a CU (tiles of 32 keys) changed nothing there.
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
        if (l != l) break;                                   // the whole row is NaN already
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

// MB: 16-row blocks per wave, one or two (rows_fwd() chooses): with two, every K and V fragment read from LDS serves two products.  EXACT
// (bf16, for a backward pass): what rounding p left over goes through the second product too, so that o, and delta with it, does not carry that
// rounding into the gradients (without it 4093 causal rows take 2 us of 256 less, and dq of short scenes is off by 0.25 % instead of 0.24).
template <typename T, int DP, int BN, int MB, bool CAP, int AX, bool EXACT>
__global__ __launch_bounds__(256, MB == 2 ? 2 : 3) void scene_attn_fwd_kernel(const SceneAttnArgs A) {
    using X = Tr<T>;
    using L = Tile<T, DP>;
    constexpr int NF = DP / X::KD, NB = BN / 16, DB = DP / 16, PB = X::KB / 16, NC = BN * L::NCH, ROWS = 64 * MB;
    static_assert(BN % X::KB == 0, "tile");
    __shared__ u32x4 sk[2][NC], sv[2][NC];
    __shared__ __attribute__((aligned(16))) float sp[2][AX ? AX : 1][BN];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const int kvh = (int)(blockIdx.x % A.KV), both = A.KV * A.key_parts, part = (int)(blockIdx.x / A.KV % A.key_parts);
    const int tiles = gridDim.x / both;
    const int64_t R = (int64_t)A.nq * A.G, r0 = (int64_t)(tiles - 1 - snake(blockIdx.x / both, tiles, max(CUS / both, 1))) * ROWS;
    const Score<CAP, AX, sizeof(T) == 4> S(A);
    constexpr bool PLAIN = !CAP && AX == 0;                 // scores stay raw until the exponent: 2^(raw k - base) in one fma
    const bool flip = PLAIN && A.scale < 0.f;               // their maximum then needs k >= 0: the sign goes to q
    const float k = flip ? -S.k : S.k;

    // the keys of the workgroup's rows; the first two tiles are on their way before anything else is read
    const int qa = row_of(r0, A.G), qb = row_of(min(r0 + ROWS, R) - 1, A.G);
    int tlo = uniform(max(A.row_lo[qa], 0)), thi = uniform(min(A.row_hi[qb], A.nk));
    if (A.key_parts > 1) key_part<BN>(tlo, thi, part, A.key_parts);
    const T *K = reinterpret_cast<const T *>(A.k) + kvh * A.k_hs, *V = reinterpret_cast<const T *>(A.v) + kvh * A.v_hs;
    const bool even = A.k_vec == 16 && A.v_vec == 16 && short_rows(A.k_rs, BN, sizeof(T)) && short_rows(A.v_rs, BN, sizeof(T));
    Stage<T, DP, BN, 256> tk, tv;
    tk.offsets([&](int r) { return (uint32_t)(r * A.k_rs * sizeof(T)); }, A.D);
    tv.offsets([&](int r) { return (uint32_t)(r * A.v_rs * sizeof(T)); }, A.D);
    auto issue = [&](int kb, int buf) {                     // keys behind the last one: the last one again, masked below
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

    RowState s[MB];
    typename X::frag qf[MB][NF];
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        s[b] = row_state(A, kvh, r0 + (w * MB + b) * 16 + c, R);
        const T *Q = reinterpret_cast<const T *>(A.q) + s[b].row * A.q_rs + s[b].head * A.q_hs;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            u32x4 v = load_chunk<T>(Q, f * X::KD + g * X::CH, A.D, A.q_vec);
            if (flip) v ^= sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
            qf[b][f] = as_frag<T>(v);
        }
    }
    // the keys of this wave's rows, and those that all of them see
    const int wlo = uniform(__shfl(s[0].lo, 0)), whi = uniform(__shfl(s[MB - 1].hi, 15));
    const int alo = uniform(__shfl(s[MB - 1].lo, 15)), ahi = uniform(__shfl(s[0].hi, 0));
    f32x4 o[MB][DB];
    float m[MB], l[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        m[b] = NEG_INF;
        l[b] = 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[b][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    int buf = 0;
    for (int kb = tlo; kb < thi; kb += BN, buf ^= 1) {
        landed();
        __syncthreads();                                    // this tile is in LDS, and nobody reads the other one any more
        if (kb > tlo && kb + BN < thi) issue(kb + BN, buf ^ 1);
        if (kb >= whi || kb + BN <= wlo) continue;
        f32x4 x[MB][NB];
        float top[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) top[b] = NEG_INF;
        auto products = [&](int n) {
#pragma unroll
            for (int b = 0; b < MB; ++b) x[b][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const typename X::frag a = frag_rows<T, DP>(sk[buf], n * 16, f, lane);
#pragma unroll
                for (int b = 0; b < MB; ++b) x[b][n] = mma(a, qf[b][f], x[b][n]);
            }
        };
        auto scores = [&](int n) {
            f32x4 px = {}, py = {}, pz = {};
            if constexpr (AX > 0) read_positions<AX>(sp[buf], n * 16 + 4 * g, px, py, pz);
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                if constexpr (!PLAIN) S.template apply<1>(&x[b][n]);
                if constexpr (AX > 0) x[b][n] -= s[b].slope * S.dist4(s[b].pos, px, py, pz);
            }
        };
        if (kb >= alo && kb + BN <= ahi) {                  // every row of the wave sees all of it: no branches between the products
#pragma unroll
            for (int n = 0; n < NB; ++n) products(n);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                scores(n);
#pragma unroll
                for (int b = 0; b < MB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top[b] = fmaxf(top[b], x[b][n][i]);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const int k0 = kb + n * 16;
                if (k0 >= whi || k0 + 16 <= wlo) {
#pragma unroll
                    for (int b = 0; b < MB; ++b) x[b][n] = f32x4{NEG_INF, NEG_INF, NEG_INF, NEG_INF};
                    continue;
                }
                products(n);
                scores(n);
#pragma unroll
                for (int b = 0; b < MB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = k0 + 4 * g + i;
                        x[b][n][i] = key >= s[b].lo && key < s[b].hi ? x[b][n][i] : NEG_INF;
                        top[b] = fmaxf(top[b], x[b][n][i]);
                    }
            }
        }
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            top[b] = group_max(top[b]);
            if constexpr (PLAIN) top[b] = top[b] == NEG_INF ? NEG_INF : top[b] * k;
            if (__any(top[b] > m[b])) {                     // a new maximum somewhere in the block: later tiles rarely bring one
                const float nm = fmaxf(top[b], m[b]), corr = exp2_(m[b] - (nm == NEG_INF ? 0.f : nm));
                m[b] = nm;
                l[b] *= corr;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[b][d] *= corr;
            }
            const float base = m[b] == NEG_INF ? 0.f : m[b];
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[b][n][i] = exp2_(PLAIN ? x[b][n][i] * k - base : x[b][n][i] - base);
                    sum += x[b][n][i];
                }
            l[b] += sum;
        }
#pragma unroll
        for (int j = 0; j < NB / PB; ++j) {
            const int k0 = kb + j * X::KB;
            if (MB == 1 && (k0 >= whi || k0 + X::KB <= wlo)) continue;
            typename X::frag p[MB], rest[MB];
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                p[b] = pack_p(&x[b][j * PB], T());
                if constexpr (EXACT) rest[b] = pack_rest(&x[b][j * PB], p[b]);
            }
            constexpr int DU = DB % 2 == 0 ? 2 : 1;         // EXACT: two accumulators in turn, so that no product waits for the one before it
#pragma unroll
            for (int d = 0; d < DB; d += DU) {
                typename X::frag a[DU];
#pragma unroll
                for (int u = 0; u < DU; ++u) a[u] = frag_cols<DP>(sv[buf], j * X::KB, d + u, lane, T());
#pragma unroll
                for (int u = 0; u < DU; ++u)
#pragma unroll
                    for (int b = 0; b < MB; ++b) o[b][d + u] = mma(a[u], p[b], o[b][d + u]);
                if constexpr (EXACT) {
#pragma unroll
                    for (int u = 0; u < DU; ++u)
#pragma unroll
                        for (int b = 0; b < MB; ++b) o[b][d + u] = mma(a[u], rest[b], o[b][d + u]);
                }
            }
        }
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        const int64_t r = r0 + (w * MB + b) * 16 + c, item = (int64_t)s[b].row * A.H + s[b].head;
        if (A.key_parts > 1) {
            const float sum = group_sum(l[b]);
            if (r < R) {
#pragma unroll
                for (int d = 0; d < DB; ++d) store4(A.part + (item * A.key_parts + part) * A.D, o[b][d], d * 16 + g * 4, A.D, A.D % 4 == 0);
                if (g == 0) {
                    A.stat[(item * A.key_parts + part) * 2] = m[b];
                    A.stat[(item * A.key_parts + part) * 2 + 1] = sum;
                }
            }
            continue;
        }
        const float sum = group_sum(l[b]), inv = sum == 0.f ? 0.f : 1.f / sum;
        bool fine = finite_(sum);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[b][d][i] *= inv;
                fine = fine && finite_(o[b][d][i]);
            }
        if (r < R) {
            const int64_t at = item * A.D;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                store4(reinterpret_cast<T *>(A.out) + at, o[b][d], d * 16 + g * 4, A.D, A.o_vec != 0);
                if (A.o32) store4(A.o32 + at, o[b][d], d * 16 + g * 4, A.D, A.o_vec != 0);
            }
            if (A.lse && g == 0) A.lse[kvh * R + r] = sum == 0.f ? 0.f : m[b] + log2_(sum);
        }
        uint64_t bad = __ballot(!fine && r < R);
        while (bad) {                                       // wave-uniform; the same row may be named by several lane groups
            const int src = __builtin_ctzll(bad) & 15;
            bad &= ~(0x0001000100010001ull << src);
            const int64_t rr = r - c + src;
            row_slow<T>(A, kvh, row_state(A, kvh, rr, R), rr, R);
        }
    }
}

// (row, head) pairs from their parts, 32 lanes each, four columns a lane
template <typename T> __global__ __launch_bounds__(256) void scene_attn_fwd_join_kernel(const SceneAttnArgs A) {
    const int lane = threadIdx.x & 63, P = A.key_parts, d = (lane & 31) * 4, vec = A.D % 4 == 0 ? 16 : 4;
    const int64_t items = (int64_t)A.nq * A.H, R = (int64_t)A.nq * A.G, own = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), item = min(own, items - 1);
    const float *stat = A.stat + item * P * 2, *part = A.part + item * P * A.D;
    float m = NEG_INF, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < P; ++i) m = fmaxf(m, stat[2 * i]);
    const float base = m == NEG_INF ? 0.f : m;
    for (int i = 0; i < P; ++i) {
        const float f = exp2_(stat[2 * i] - base);
        l += f * stat[2 * i + 1];
        o += f * __builtin_bit_cast(f32x4, load_chunk<float>(part + (int64_t)i * A.D, d, A.D, vec));
    }
    o *= l == 0.f ? 0.f : 1.f / l;
    const int64_t row = item / A.H;
    const int head = (int)(item - row * A.H), kvh = head / A.G;
    const int64_t r = row * A.G + head - kvh * A.G;
    if (own < items) {
        store4(reinterpret_cast<T *>(A.out) + item * A.D, o, d, A.D, A.o_vec != 0);
        if (A.o32) store4(A.o32 + item * A.D, o, d, A.D, A.o_vec != 0);
        if (A.lse && d == 0) A.lse[kvh * R + r] = l == 0.f ? 0.f : m + log2_(l);
    }
    const bool fine = own >= items || (finite_(l) && finite_(o[0]) && finite_(o[1]) && finite_(o[2]) && finite_(o[3]));
    const uint64_t bad = __ballot(!fine);
    for (int h = 0; h < 2; ++h)                              // the wave's two pairs
        if (bad >> (32 * h) & 0xffffffffull) row_slow<T>(A, __shfl(kvh, 32 * h), row_state(A, __shfl(kvh, 32 * h), __shfl(r, 32 * h), R), __shfl(r, 32 * h), R);
}

template <typename T, int DP, int BN, int MB, bool CAP, int AX> hipError_t launch_fwd(const SceneAttnArgs &A, hipStream_t st) {
    const int64_t tiles = ((int64_t)A.nq * A.G + 64 * MB - 1) / (64 * MB);
    const dim3 grid((unsigned)(tiles * A.KV * A.key_parts));
    constexpr bool EXACT = sizeof(T) == 2;                 // fp32 rounds no p
    if (EXACT && A.o32) hipLaunchKernelGGL((scene_attn_fwd_kernel<T, DP, BN, MB, CAP, AX, EXACT>), grid, dim3(256), 0, st, A);
    else hipLaunchKernelGGL((scene_attn_fwd_kernel<T, DP, BN, MB, CAP, AX, false>), grid, dim3(256), 0, st, A);
    if (A.key_parts > 1) hipLaunchKernelGGL((scene_attn_fwd_join_kernel<T>), dim3((unsigned)(((int64_t)A.nq * A.H + 7) / 8)), dim3(256), 0, st, A);
    return hipGetLastError();
}
// Workgroups of a kernel that a CU holds at once (its registers and LDS)
template <void (*KERNEL)(const SceneAttnArgs)> int held() {
    static const int n = [] {
        int v = 0;
        return hipOccupancyMaxActiveBlocksPerMultiprocessor(&v, KERNEL, 256, 0) == hipSuccess && v > 0 ? v : 1;
    }();
    return n;
}
// Two blocks of 16 rows a wave read K and V from LDS half as often but leave a CU with fewer workgroups, of 128 rows instead of 64.  Worth it where the
// products weigh more than the scores' vector work (cap, distance), the more so the wider a head (the condition below), and
// - where rows see alike numbers of keys, if a CU gets through its workgroups in fewer rounds; in as many rounds only where it holds three of them at
//   once (with two the waits show) and has more than three of 64 rows to do.  bf16, 8 heads to 2, all seen, us with one block and with two, at (tiles of
//   128 rows, for all heads) 320, 400, 512, 544, 672, 768, 896, 1024, 1152:
//       width 64 (a CU holds 5 and 3): 119 133, 159 153, 214 198, 288 261, 392 325, 455 380, 599 593, 774 694, 990 893
//       width 96 (3 and 2):            131 147, 255 187, 339 233, 369 430, 506 530, 596 607, 935 750, 1096 878, 1324 1371;  capped 187 234, 337 293, 438 382,
//                                      511 635, 729 788, 852 906, 1203 1272, 1471 1451, 1910 2108
//       width 128 (2 and 2):           230 182, 304 231, 391 290, 579 548, 751 671, 869 765, 1350 934, 1567 1083, 2171 1743;  capped 294 265, 404 329,
//                                      519 416, 742 763, 993 936, 1139 1074, 1678 1401, 1984 1603, 2691 2472
// - where they see unlike numbers, from 768 workgroups on: short tiles fill up behind long ones.  Causal, 8192 rows: width 64 126 164, 96 178 205, 128 227 258;
//   16384: 401 361, 571 502, 812 631
// What the condition on the width leaves out, 16384 rows, all seen: width 64, cap 1184 1202;  96, cap and an axis 1582 1617;  128, cap and three axes 2520 2618.
template <typename T, int DP, int BN, bool CAP, int AX> hipError_t rows_fwd(const SceneAttnArgs &A, hipStream_t st) {
    if constexpr (sizeof(T) == 2 && DP >= 64 && (CAP ? 2 : 0) + (AX > 1 ? 2 : AX) < DP / 32) {
        const int64_t R = (int64_t)A.nq * A.G, two = (R + 127) / 128 * A.KV, one = (R + 63) / 64 * A.KV;
        const int h1 = A.o32 ? held<scene_attn_fwd_kernel<T, DP, BN, 1, CAP, AX, true>>() : held<scene_attn_fwd_kernel<T, DP, BN, 1, CAP, AX, false>>();
        const int h2 = A.o32 ? held<scene_attn_fwd_kernel<T, DP, BN, 2, CAP, AX, true>>() : held<scene_attn_fwd_kernel<T, DP, BN, 2, CAP, AX, false>>();
        const int64_t n1 = (one + CUS - 1) / CUS, n2 = (two + CUS - 1) / CUS, rounds1 = (n1 + h1 - 1) / h1, rounds2 = (n2 + h2 - 1) / h2;
        if (A.uneven ? two >= 768 : rounds2 < rounds1 || (rounds2 == rounds1 && h2 >= 3 && n1 > 3)) return launch_fwd<T, DP, BN, 2, CAP, AX>(A, st);
    }
    return launch_fwd<T, DP, BN, 1, CAP, AX>(A, st);
}
template <typename T, int DP, int BN> hipError_t pick_fwd(const SceneAttnArgs &A, hipStream_t st) {
    if (A.cap > 0.f) return A.axes == 0 ? rows_fwd<T, DP, BN, true, 0>(A, st) : A.axes == 1 ? rows_fwd<T, DP, BN, true, 1>(A, st) : rows_fwd<T, DP, BN, true, 3>(A, st);
    return factor_last(A) ? rows_fwd<T, DP, BN, false, 0>(A, st) : A.axes <= 1 ? rows_fwd<T, DP, BN, false, 1>(A, st) : rows_fwd<T, DP, BN, false, 3>(A, st);
}

}  // namespace sattn

// one object file per type (the Makefile compiles this source twice)
#ifdef SCENE_ATTN_BF16
extern "C" hipError_t dn_scene_attn_fwd_bf16(const SceneAttnArgs *A, hipStream_t st) {
    using namespace sattn;
    const int D = A->D;
    return D <= 32 ? pick_fwd<bf16, 32, 64>(*A, st) : D <= 64 ? pick_fwd<bf16, 64, 64>(*A, st) : D <= 96 ? pick_fwd<bf16, 96, 64>(*A, st) : pick_fwd<bf16, 128, 64>(*A, st);
}
#else
extern "C" hipError_t dn_scene_attn_fwd_f32(const SceneAttnArgs *A, hipStream_t st) {
    using namespace sattn;
    const int D = A->D;
    return D <= 16 ? pick_fwd<float, 16, 64>(*A, st) : D <= 32 ? pick_fwd<float, 32, 64>(*A, st) : D <= 48 ? pick_fwd<float, 48, 32>(*A, st)
         : D <= 64 ? pick_fwd<float, 64, 32>(*A, st) : D <= 96 ? pick_fwd<float, 96, 32>(*A, st) : pick_fwd<float, 128, 32>(*A, st);
}
// whether rows see unlike numbers of keys
extern "C" int dn_scene_attn_uneven(int64_t most, int64_t mean) { return 3 * mean < 2 * most; }
// Parts of the keys of a row tile, forward and dq, where there are few tiles: none below 128 of the keys that a row sees (most), and as many as give the
// chip's CUs three workgroups each (what their registers and LDS hold) - four where rows see unlike numbers of keys (mean far below most): then the
// longest tile is what the rest waits for.  4096 causal bf16 rows of 8 heads: 102 us in one part, 66 + 8 to join in two; seeing all keys: 92 and 121.
// The least part, 1000 fp32 rows and keys, 4 heads of 72 to one: 42 us with 256 keys, 37 with 128 (512 keys, 25 and 18), 33 with 64; in bf16 18.4,
// 18.8 and 18.3 (512 keys of 8 heads of 32: 11.8, 10.7 and 13.0: the join's share grows).
extern "C" int dn_scene_attn_key_parts(int64_t nq, int KV, int G, int64_t most, int64_t mean) {
    const int64_t tiles = (nq * G + 63) / 64 * KV, want = tiles ? (dn_scene_attn_uneven(most, mean) ? 1024 : 768) / tiles : 1, parts = want < most / 128 ? want : most / 128;
    return (int)(parts < 1 ? 1 : parts < 8 ? parts : 8);
}
#endif
