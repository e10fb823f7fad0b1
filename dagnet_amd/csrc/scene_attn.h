// Attention over the rows of a scene: what the forward, backward and step kernels share.
//
// Row i (a query row) of head h sees the keys j of one interval, row_lo[i] <= j < row_hi[i]; both bounds never decrease with i.  Scenes
// (a batch is packed scene after scene), causal order by time step and an observed prefix are all intervals of that kind, so the
// kernels know nothing of scenes: a tile of rows walks the keys from its first row's lo to its last row's hi and masks by interval, and
// small scenes share a tile.
//     x_ij = cap tanh(scale q_i.k_j / cap) - slope_h |pos_i - pos_j|,   p_i = softmax_j x_ij,   o_i = sum_j p_ij v_j
// Softmax statistics are kept in base 2: x / ln 2, one v_exp_f32 per score.
//
// Heads that share keys (group size G = heads / kv heads) are rows of one tile: packed row r of kv head c is row r / G of head
// c G + r % G.  K and V are then read once for the whole group, and gradients of shared keys need no sum over heads afterwards.
//
// Matrix layout (v_mfma 16x16): lane l = 16 g + c holds column c of the accumulator, rows 4 g .. 4 g + 3.  The scores are computed
// transposed (keys along the rows, query rows along the columns), so a lane holds 4 consecutive keys of ONE query row: statistics are
// lane-local but for two shuffles, and the accumulator registers already are the second product's operand (its contraction runs over
// the same keys in the same order on both sides; which key stands at which k does not matter).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

struct SceneAttnArgs {
    const void *q, *k, *v, *dout;              // dout: gradient of the output (backward)
    void *out, *dq, *dk, *dv;
    float *lse, *o32, *delta, *dsl;            // lse, delta, dsl: [kv heads][nq * G]; o32: [nq][H][D], the unrounded output (read back by the backward)
    const float *slopes, *qpos, *kpos;         // [H]; [nq][axes], [nk][axes]
    const int32_t *row_lo, *row_hi;            // [nq]
    const int32_t *key_lo, *key_hi;            // [nk]: rows that see a key (backward)
    int64_t q_rs, q_hs, k_rs, k_hs, v_rs, v_hs, do_rs, do_hs;      // element strides of rows and heads (out, dq, dk, dv: contiguous)
    int32_t nq, nk, H, KV, G, D, axes;
    float scale, cap;
    int32_t parts;                             // of the rows in the dk / dv kernel; part: [parts][dk, dv][nk][KV][D]
    float *part;
    int32_t q_vec, k_vec, v_vec, do_vec, o32_vec;   // bytes per load that strides, base and width allow: 16, 8 or the element
    int32_t o_vec;                                 // results are stored four at a time
};

namespace sattn {

typedef __bf16 bf16;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEG_INF = -__builtin_inff();

// Chunk: 16 bytes of a row.  Frag: one chunk per lane, 4 lane groups = KD consecutive columns of a row, one k-slice of a product.
template <typename T> struct Tr;
template <> struct Tr<float> {
    typedef f32x4 frag;
    static constexpr int CH = 4, KD = 16, KB = 16;      // elements per chunk, columns per frag, keys per frag of the second product
};
template <> struct Tr<bf16> {
    typedef bf16x8 frag;
    static constexpr int CH = 8, KD = 32, KB = 32;
};

__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float rcp_(float x) { return __builtin_amdgcn_rcpf(x); }

// elements [d, d + CH) of a row of D elements; zeros behind D.  vec: bytes per load (16: the whole chunk, then D % CH == 0)
template <typename T> __device__ __forceinline__ u32x4 load_chunk(const T *p, int d, int D, int vec) {
    u32x4 r = {0u, 0u, 0u, 0u};
    if (d >= D) return r;
    if (vec == 16) return *reinterpret_cast<const u32x4 *>(p + d);
    constexpr int CH = Tr<T>::CH;
    if (vec == 8) {
        const u32x2 a = *reinterpret_cast<const u32x2 *>(p + d);
        r[0] = a[0]; r[1] = a[1];
        if (d + CH / 2 < D) {
            const u32x2 b = *reinterpret_cast<const u32x2 *>(p + d + CH / 2);
            r[2] = b[0]; r[3] = b[1];
        }
        return r;
    }
    union { T e[CH]; u32x4 v; } x;
    x.v = r;
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (d + i < D) x.e[i] = p[d + i];
    return x.v;
}

template <typename T> __device__ __forceinline__ typename Tr<T>::frag as_frag(u32x4 v) {
    union { u32x4 v; typename Tr<T>::frag f; } x;
    x.v = v;
    return x.f;
}

// Rows of a tile in LDS: NCH chunks each, chunk c of row r at slot c ^ swz(r), so that 16 lanes reading one chunk column of 16 rows
// spread over the banks (rows of less than 128 bytes share a bank line: those rows keep one swizzle).
template <typename T, int DP> struct Tile {
    static constexpr int NCH = DP / Tr<T>::CH;
    static __device__ __forceinline__ int swz(int r) { return NCH % 8 == 0 ? (r & 7) : NCH > 8 ? (r & 3) : ((r / (8 / NCH)) & (NCH - 1)); }
    static __device__ __forceinline__ int slot(int r, int c) { return r * NCH + (c ^ swz(r)); }
};

// Fills a tile of ROWS rows with the rows row(r) points to (columns behind D: anything finite that the row holds - the other operand is 0
// there, or the result is not stored).  vec 16: straight into LDS, 64 lanes x 16 bytes an instruction, the swizzle applied to the
// source; nothing waits until landed().  Else through registers, done on return.
template <typename T, int DP, int ROWS, int NT, typename Row> __device__ __forceinline__ void stage(u32x4 *tile, Row row, int D, int vec) {
    using L = Tile<T, DP>;
    constexpr int NC = ROWS * L::NCH, PER = (NC + NT - 1) / NT;
    static_assert(NC % 64 == 0, "whole waves");
    typedef __attribute__((address_space(3))) void *lp;
    typedef const __attribute__((address_space(1))) void *gp;
    const int lane = threadIdx.x & 63, w0 = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63);
    if (vec == 16) {
        const int last = (D - 1) / Tr<T>::CH;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int s0 = i * NT + w0;
            if (NC % NT == 0 || s0 < NC) {
                const int s = s0 + lane, r = s / L::NCH, c = (s % L::NCH) ^ L::swz(r);
                __builtin_amdgcn_global_load_lds((gp)(row(r) + min(c, last) * Tr<T>::CH), (lp)(tile + s0), 16, 0, 0);
            }
        }
    } else {
#pragma unroll 1
        for (int s = threadIdx.x; s < NC; s += NT) {
            const int r = s / L::NCH, c = (s % L::NCH) ^ L::swz(r);
            tile[s] = load_chunk<T>(row(r), c * Tr<T>::CH, D, vec);
        }
    }
}
// this wave's part of every stage() so far is in LDS (a barrier then says so of the workgroup's)
__device__ __forceinline__ void landed() { __builtin_amdgcn_s_waitcnt(0x0f70); }      // vmcnt(0)

// A operand of the first product: row r0 + c of a tile, columns kk KD + ..
template <typename T, int DP> __device__ __forceinline__ typename Tr<T>::frag frag_rows(const u32x4 *t, int r0, int kk, int lane) {
    return as_frag<T>(t[Tile<T, DP>::slot(r0 + (lane & 15), kk * 4 + (lane >> 4))]);
}

// A operand of the second product: the transposed tile, columns d = 16 db + c, rows r0 + (what the scores' registers hold: 4 g + i of
// one block of 16 rows, or of two for 16-bit types).  16-bit types: ds_read_b64_tr_b16 hands lane c of a group of 16 column c of the
// 4 x 16 block whose rows the group's lanes address four by four.
template <int DP> __device__ __forceinline__ f32x4 frag_cols(const u32x4 *t, int r0, int db, int lane, float) {
    const float *f = reinterpret_cast<const float *>(t);
    f32x4 a;
    const int c = lane & 15, r = r0 + 4 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = f[Tile<float, DP>::slot(r + i, db * 4 + (c >> 2)) * 4 + (c & 3)];
    return a;
}
template <int DP> __device__ __forceinline__ bf16x8 frag_cols(const u32x4 *t, int r0, int db, int lane, bf16) {
    typedef __attribute__((address_space(3))) s16x4 *lp;
    const int c = lane & 15, r = r0 + 4 * (lane >> 4) + (c >> 2);
    union { s16x4 h[2]; bf16x8 f; } x;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const char *p = reinterpret_cast<const char *>(t + Tile<bf16, DP>::slot(r + 16 * i, db * 2 + ((c & 3) >> 1))) + (c & 1) * 8;
        x.h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p);
    }
    return x.f;
}

// B operand of the second product from score-shaped registers; P and dS are rounded to the inputs' type here and nowhere else
__device__ __forceinline__ f32x4 pack_p(const f32x4 *p, float) { return p[0]; }
__device__ __forceinline__ bf16x8 pack_p(const f32x4 *p, bf16) {
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) { r[i] = (bf16)p[0][i]; r[4 + i] = (bf16)p[1][i]; }
    return r;
}

// what that rounding left over, rounded in turn: p to 16 bits through two products
__device__ __forceinline__ bf16x8 pack_rest(const f32x4 *p, bf16x8 hi) {
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) { r[i] = (bf16)(p[0][i] - (float)hi[i]); r[4 + i] = (bf16)(p[1][i] - (float)hi[4 + i]); }
    return r;
}
__device__ __forceinline__ f32x4 pack_rest(const f32x4 *, f32x4 hi) { return hi; }      // fp32 rounds nothing: never used

// tanh to about 1 ulp of fp32: near zero the odd rational [7/6] from the continued fraction x / (1 + x^2 / (3 + x^2 / (5 + ...)))
// (its next term is below 2^-27 for |x| <= 1), else 1 - 2 / (1 + e^2x), which loses nothing there.
__device__ __forceinline__ float tanh_(float x) {
    const float a = fabsf(x);
    const float e = exp2_(a * (2.f * LOG2E));
    const float far = 1.f - 2.f * rcp_(1.f + e);
    const float s = x * x;
    const float n = a * (135135.f + s * (17325.f + s * (378.f + s)));
    const float d = 135135.f + s * (62370.f + s * (3150.f + s * 28.f));
    const float near = n * rcp_(d);
    return copysignf(a < 1.f ? near : far, x);
}

__device__ __forceinline__ float distance(int axes, const float *a, const float *b) {
    const float x = a[0] - b[0];
    if (axes == 1) return fabsf(x);
    const float y = a[1] - b[1];
    float s = x * x + y * y;
    if (axes == 3) {
        const float z = a[2] - b[2];
        s += z * z;
    }
    return __builtin_amdgcn_sqrtf(s);
}

__device__ __forceinline__ bool finite_(float x) { return fabsf(x) < __builtin_inff(); }
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16 x) { return (float)x; }

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// over the four lane groups of one column
__device__ __forceinline__ float group_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float group_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Row c of the wave (all four lane groups hold the same), as the kernels keep it per lane.
struct RowState {
    int row, head, lo, hi;
    float slope, pos[3];
};

__device__ __forceinline__ RowState row_state(const SceneAttnArgs &A, int kvh, int64_t r, int64_t R) {
    RowState s;
    const int64_t rr = r < R ? r : R - 1;
    s.row = (int)(rr / A.G);
    s.head = kvh * A.G + (int)(rr - (int64_t)s.row * A.G);
    s.lo = max(A.row_lo[s.row], 0);
    s.hi = min(A.row_hi[s.row], A.nk);
    s.slope = A.axes ? A.slopes[s.head] * LOG2E : 0.f;
    s.pos[0] = s.pos[1] = s.pos[2] = 0.f;
    const float *p = A.qpos + (int64_t)s.row * A.axes;
    if (A.axes > 0) s.pos[0] = p[0];
    if (A.axes > 1) s.pos[1] = p[1];
    if (A.axes > 2) s.pos[2] = p[2];
    return s;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Coordinate a of a tile's keys, loaded by the first lanes; missing axes are 0.
template <int AX, int N> struct KeyPos {
    float r[AX ? AX : 1];
    __device__ __forceinline__ void fetch(const SceneAttnArgs &A, const float *kpos, int key) {
        if constexpr (AX > 0)
            if (threadIdx.x < N) {
#pragma unroll
                for (int a = 0; a < AX; ++a) r[a] = a < A.axes ? kpos[(int64_t)key * A.axes + a] : 0.f;
            }
    }
    __device__ __forceinline__ void put(float (*s)[N]) const {
        if constexpr (AX > 0)
            if (threadIdx.x < N) {
#pragma unroll
                for (int a = 0; a < AX; ++a) s[a][threadIdx.x] = r[a];
            }
    }
};

// Scores in base 2 from raw products, the constants of one launch folded together.  CAP and AX (0, 1, or 3 for two and three
// coordinates) are compiled in: the kernels are bound by vector instructions per score, not by the products.
//   cap: t = tanh(raw scale / cap) = 1 - 2 r with r = 1 / (1 + e^2z); x = cap t.  In fp32 near zero through tanh_() (1 - 2 r is off by 2^-24 there
//   whatever t is); for bf16 that is far below what the operands' type can tell.
template <typename T, bool CAP, int AX> struct Score {
    float k, cap2, arg;
    __device__ __forceinline__ Score(const SceneAttnArgs &A) {
        k = A.scale * LOG2E;
        cap2 = A.cap * LOG2E;
        arg = CAP ? (sizeof(T) == 4 ? A.scale / A.cap : 2.f * LOG2E * A.scale / A.cap) : 0.f;
    }
    // x in base 2; t: the tanh (for its derivative)
    __device__ __forceinline__ float value(float raw, float &t) const {
        if constexpr (!CAP) return raw * k;
        else {
            if constexpr (sizeof(T) == 4) t = tanh_(raw * arg);
            else t = 1.f - 2.f * rcp_(1.f + exp2_(raw * arg));
            return cap2 * t;
        }
    }
    static __device__ __forceinline__ float dist(const float *a, float bx, float by, float bz) {
        const float x = a[0] - bx;
        if constexpr (AX == 1) return fabsf(x);
        const float y = a[1] - by, z = a[2] - bz;
        return __builtin_amdgcn_sqrtf(x * x + y * y + z * z);
    }
};

// the same with everything read at run time (the slow forms and the step kernel's launch-time choices)
__device__ __forceinline__ float score2(const SceneAttnArgs &A, float raw, float inv_cap, float slope2, const float *qpos, const float *kpos) {
    float x = raw * A.scale;
    if (A.cap > 0.f) x = A.cap * tanh_(x * inv_cap);
    x *= LOG2E;
    if (A.axes) x -= slope2 * distance(A.axes, qpos, kpos);
    return x;
}

// 4 consecutive values of a row, rounded once
template <typename T> __device__ __forceinline__ void store4(T *p, f32x4 v, int d, int D, bool vec) {
    if (vec) {
        if (d < D) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4 *>(p + d) = v;
            else {
                bf16x4 h;
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = (bf16)v[i];
                *reinterpret_cast<bf16x4 *>(p + d) = h;
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (d + i < D) p[d + i] = (T)v[i];
}

}  // namespace sattn
