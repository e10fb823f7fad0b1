// Scene attention of the new rows of a step over kept keys (scene_attn.h has the mathematics and the layout): scene s keeps its keys and
// values in rows 0 .. k_len[s] - 1 of its own stretch of a cache, and all of its new rows see all of them.
//
// Few rows, many keys: the keys are read once and bound the kernel.  One workgroup takes one scene, one kv head, 16 packed rows (the new
// rows times the heads that share keys) and one split of the keys; its four waves take 32 (16-bit) or 16 (fp32) keys in turn, K straight
// from memory into the first product's operand, V through a wave's own stretch of LDS for the transposed one.  The splits' partial
// outputs, maxima and sums meet in scene_attn_join_kernel.
//
// Bound by the cache's bytes: bf16, 4 sequences of 60 000 to 131 071 keys, 4 key heads of 128, one row each: 184 us for 887 MB, 4.8 TB/s - what a large copy
// reaches.  256 scenes of ten rows over 280 to 2000 keys (8 heads of 64 to 2, cap, three axes): 72 us for 139 MB; there the blocks' vector work counts
// (58 instructions a score, issuing in 59 % of the busy clocks).
#include "scene_attn.h"
#include "scene_attn_step.h"
#include <algorithm>

namespace sattn {

template <typename T, int DP, bool CAP, int AX> __global__ __launch_bounds__(256) void scene_attn_step_kernel(const SceneStepArgs A) {
    using X = Tr<T>;
    using L = Tile<T, DP>;
    constexpr int NF = DP / X::KD, DB = DP / 16, PB = X::KB / 16, NC = X::KB * L::NCH, PER = NC / 64;
    constexpr bool PLAIN = !CAP && AX == 0;
    static_assert(NC % 64 == 0 && X::KB <= 64, "tile");
    __shared__ u32x4 sv[4][NC];
    __shared__ __attribute__((aligned(16))) float sp[4][AX ? AX : 1][X::KB];
    __shared__ float sm[4][16], sl[4][16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    int64_t id = blockIdx.x;
    const int kvh = (int)(id % A.a.KV);
    id /= A.a.KV;
    const int split = (int)(id % A.splits);
    id /= A.splits;
    const int cb = (int)(id % A.cblocks), sc = (int)(id / A.cblocks);
    const int q0 = max(A.q_ptr[sc], 0), q1 = min(A.q_ptr[sc + 1], A.a.nq);
    const int64_t n = (int64_t)(q1 - q0) * A.a.G;
    if ((int64_t)cb * 16 >= n) return;                              // the whole workgroup
    const int len = min(max(A.k_len[sc], 0), A.room);
    const int per = (int)((((int64_t)len + A.splits - 1) / A.splits + 4 * X::KB - 1) / (4 * X::KB)) * (4 * X::KB);   // whole rounds of the four waves
    const int ka = (int)min((int64_t)split * per, (int64_t)len), kz = (int)min((int64_t)ka + per, (int64_t)len);
    const Score<CAP, AX, sizeof(T) == 4> S(A.a);
    const bool flip = PLAIN && A.a.scale < 0.f;
    const float k = flip ? -S.k : S.k;
    const T *K = reinterpret_cast<const T *>(A.a.k) + sc * A.k_ss + kvh * A.a.k_hs, *V = reinterpret_cast<const T *>(A.a.v) + sc * A.v_ss + kvh * A.a.v_hs;
    const float *kpos = A.a.kpos + (int64_t)sc * A.room * A.a.axes;

    u32x4 rk[PB][NF], rv[PER];
    float rp[AX ? AX : 1];
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
        if constexpr (AX > 0) {
            const float *p = kpos + (int64_t)min(k0 + (lane & (X::KB - 1)), len - 1) * A.a.axes;
#pragma unroll
            for (int a = 0; a < AX; ++a) rp[a] = a < A.a.axes ? p[a] : 0.f;
        }
    };
    int k0 = ka + w * X::KB;
    if (k0 < kz) fetch(k0);

    const int64_t pr = min((int64_t)cb * 16 + c, n - 1);
    const int row = q0 + (int)(pr / A.a.G), head = kvh * A.a.G + (int)(pr % A.a.G);
    const float slope = AX && A.a.axes ? A.a.slopes[head] * LOG2E : 0.f;
    float qpos[3];
#pragma unroll
    for (int a = 0; a < 3; ++a) qpos[a] = a < AX && a < A.a.axes ? A.a.qpos[(int64_t)row * A.a.axes + a] : 0.f;
    const T *Q = reinterpret_cast<const T *>(A.a.q) + row * A.a.q_rs + head * A.a.q_hs;
    typename X::frag qf[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        u32x4 v = load_chunk<T>(Q, f * X::KD + g * X::CH, A.a.D, A.a.q_vec);
        if (flip) v ^= sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
        qf[f] = as_frag<T>(v);
    }
    f32x4 o[DB];
    float m = NEG_INF, l = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (; k0 < kz; k0 += 4 * X::KB) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane + i * 64;
            sv[w][L::slot(e / L::NCH, e % L::NCH)] = rv[i];
        }
        if constexpr (AX > 0) {
            if (lane < X::KB) {
#pragma unroll
                for (int a = 0; a < AX; ++a) sp[w][a][lane] = rp[a];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");      // the wave's own LDS writes, before its reads across lanes
        __builtin_amdgcn_wave_barrier();
        f32x4 x[PB];
#pragma unroll
        for (int j = 0; j < PB; ++j) {
            x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < NF; ++f) x[j] = mma(as_frag<T>(rk[j][f]), qf[f], x[j]);
        }
        if (k0 + 4 * X::KB < kz) fetch(k0 + 4 * X::KB);
        if constexpr (!PLAIN) S.template apply<PB>(x);
        if constexpr (AX > 0) {
#pragma unroll
            for (int j = 0; j < PB; ++j) {
                f32x4 px = {}, py = {}, pz = {};
                read_positions<AX>(sp[w], j * 16 + 4 * g, px, py, pz);
                x[j] -= slope * S.dist4(qpos, px, py, pz);
            }
        }
        if (k0 + X::KB > kz) {
#pragma unroll
            for (int j = 0; j < PB; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[j][i] = k0 + j * 16 + 4 * g + i < kz ? x[j][i] : NEG_INF;
        }
        float top = NEG_INF;
#pragma unroll
        for (int j = 0; j < PB; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, x[j][i]);
        top = group_max(top);
        if constexpr (PLAIN) top = top == NEG_INF ? NEG_INF : top * k;
        if (__any(top > m)) {
            const float nm = fmaxf(top, m), corr = exp2_(m - (nm == NEG_INF ? 0.f : nm));
            m = nm;
            l *= corr;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= corr;
        }
        const float base = m == NEG_INF ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < PB; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[j][i] = exp2_(PLAIN ? x[j][i] * k - base : x[j][i] - base);
                sum += x[j][i];
            }
        l += sum;
        const typename X::frag p = pack_p(x, T());
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = mma(frag_cols<DP>(sv[w], 0, d, lane, T()), p, o[d]);
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // the four waves' parts: statistics first, then the outputs, rescaled, through the waves' V stretches
    l = group_sum(l);
    if (g == 0) { sm[w][c] = m; sl[w][c] = l; }
    __syncthreads();
    float *so = reinterpret_cast<float *>(&sv[0][0]);                // [4 waves][16][DP]
    static_assert(4 * NC * 4 >= 4 * 16 * DP, "LDS");
    float M = NEG_INF, sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) M = fmaxf(M, sm[i][c]);
    const float base = M == NEG_INF ? 0.f : M;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += sl[i][c] * exp2_(sm[i][c] - base);
    const float corr = exp2_(m - base);
#pragma unroll
    for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4 *>(so + (w * 16 + c) * DP + d * 16 + g * 4) = o[d] * corr;
    __syncthreads();
    if ((int64_t)cb * 16 + c >= n) return;
    const int64_t item = (int64_t)row * A.a.H + head;
    const float inv = A.splits > 1 ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int d = 0; d < DB; ++d) {                                   // every wave sums and stores its share of the columns
        if (d % 4 != w) continue;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) acc += *reinterpret_cast<const f32x4 *>(so + (i * 16 + c) * DP + d * 16 + g * 4);
        if (A.splits > 1) store4(A.part + (item * A.splits + split) * A.a.D, acc, d * 16 + g * 4, A.a.D, A.a.D % 4 == 0);
        else store4(reinterpret_cast<T *>(A.a.out) + item * A.a.D, acc * inv, d * 16 + g * 4, A.a.D, A.a.o_vec != 0);
    }
    if (A.splits > 1 && w == 0 && g == 0) {
        A.stat[(item * A.splits + split) * 2] = M;
        A.stat[(item * A.splits + split) * 2 + 1] = sum;
    }
}

// The splits of a (row, head) joined: TP threads, 32 of them over the columns (four each), the rest over the splits.  Rows that no scene owns (in front of the
// first one's, behind the last one's) have no splits and stay as they were.
template <typename T, int TP> __global__ __launch_bounds__(256) void scene_attn_join_kernel(const SceneStepArgs A) {
    constexpr int IT = 256 / TP, GR = TP / 32;
    __shared__ f32x4 so[256];
    __shared__ float sm[256 / 32], sl[256 / 32];
    const int t = threadIdx.x % TP, it = threadIdx.x / TP, d = (t % 32) * 4, gr = t / 32, D = A.a.D;
    const int64_t items = (int64_t)A.a.nq * A.a.H, item = min((int64_t)blockIdx.x * IT + it, items - 1);
    const float *stat = A.stat + item * A.splits * 2, *part = A.part + item * A.splits * D;
    const int vec = D % 4 == 0 ? 16 : 4;
    float m = NEG_INF, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i = gr; i < A.splits; i += GR) {
        const float mi = stat[2 * i], li = stat[2 * i + 1];
        const f32x4 v = __builtin_bit_cast(f32x4, load_chunk<float>(part + (int64_t)i * D, d, D, vec));
        const float nm = fmaxf(m, mi), base = nm == NEG_INF ? 0.f : nm, fa = exp2_(m - base), fb = exp2_(mi - base);
        l = l * fa + li * fb;
        o = o * fa + v * fb;
        m = nm;
    }
    so[threadIdx.x] = o;
    if (t % 32 == 0) { sm[threadIdx.x / 32] = m; sl[threadIdx.x / 32] = l; }
    __syncthreads();
    if (gr) return;
    float M = NEG_INF;
#pragma unroll
    for (int i = 0; i < GR; ++i) M = fmaxf(M, sm[it * GR + i]);
    const float base = M == NEG_INF ? 0.f : M;
    l = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < GR; ++i) {
        const float f = exp2_(sm[it * GR + i] - base);
        l += f * sl[it * GR + i];
        o += f * so[it * TP + i * 32 + t];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t row = item / A.a.H;
    const bool owned = row >= A.q_ptr[0] && row < A.q_ptr[A.scenes];
    if (owned && (int64_t)blockIdx.x * IT + it < items) store4(reinterpret_cast<T *>(A.a.out) + item * D, o * inv, d, D, A.a.o_vec != 0);
}

template <typename T, int DP, bool CAP, int AX> hipError_t launch_step(const SceneStepArgs &A, hipStream_t st) {
    const int64_t blocks = (int64_t)A.scenes * A.a.KV * A.splits * A.cblocks, items = (int64_t)A.a.nq * A.a.H;
    hipLaunchKernelGGL((scene_attn_step_kernel<T, DP, CAP, AX>), dim3((unsigned)blocks), dim3(256), 0, st, A);
    if (A.splits > 8) hipLaunchKernelGGL((scene_attn_join_kernel<T, 256>), dim3((unsigned)items), dim3(256), 0, st, A);
    else if (A.splits > 1) hipLaunchKernelGGL((scene_attn_join_kernel<T, 64>), dim3((unsigned)((items + 3) / 4)), dim3(256), 0, st, A);
    return hipGetLastError();
}
template <typename T, int DP> hipError_t pick_step(const SceneStepArgs &A, hipStream_t st) {
    const int ax = A.a.axes;
    if (A.a.cap > 0.f) return ax == 0 ? launch_step<T, DP, true, 0>(A, st) : ax == 1 ? launch_step<T, DP, true, 1>(A, st) : launch_step<T, DP, true, 3>(A, st);
    return factor_last(A.a) ? launch_step<T, DP, false, 0>(A, st) : ax <= 1 ? launch_step<T, DP, false, 1>(A, st) : launch_step<T, DP, false, 3>(A, st);
}

}  // namespace sattn

// one object file per type (the Makefile compiles this source twice)
#ifdef SCENE_ATTN_BF16
extern "C" hipError_t dn_scene_attn_step_bf16(const SceneStepArgs *A, hipStream_t st) {
    using namespace sattn;
    const int D = A->a.D;
    return D <= 32 ? pick_step<bf16, 32>(*A, st) : D <= 64 ? pick_step<bf16, 64>(*A, st) : pick_step<bf16, 128>(*A, st);
}
#else
extern "C" hipError_t dn_scene_attn_step_f32(const SceneStepArgs *A, hipStream_t st) {
    using namespace sattn;
    const int D = A->a.D;
    return D <= 16 ? pick_step<float, 16>(*A, st) : D <= 32 ? pick_step<float, 32>(*A, st) : D <= 64 ? pick_step<float, 64>(*A, st) : pick_step<float, 128>(*A, st);
}
// rows: packed rows of the largest scene; kv_scenes: scenes x kv heads.  Splits of the keys: 1536 workgroups in all - two or three full rounds of what the
// chip's 256 CUs hold at once (1024 left a third of a round at its end: 131 000 keys of 64 rows 215 us, 185 with 1536) - but none below 256 keys of the
// cache.  Several blocks of 16 rows that share keys are workgroups of their own: one workgroup for two blocks halves the reads, which
// come from L2 then, but its registers leave half as many waves (2000 keys of 256 scenes, 34 packed rows: 85 us, 72 in blocks of their own).
extern "C" void dn_scene_attn_step_shape(int64_t rows, int64_t kv_scenes, int room, int *cblocks, int *splits) {
    *cblocks = (int)((rows + 15) / 16);
    const int64_t groups = kv_scenes * *cblocks, want = (1536 + groups - 1) / groups, most = ((int64_t)room + 255) / 256;
    *splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 128));
}
#endif
