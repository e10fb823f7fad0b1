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
    // Few tiles: their long axis is cut, the parts' sums meet in a join kernel.  key_parts: of a row tile's keys (forward: part [nq H][parts][D], stat
    // [nq H][parts][2]; dq: part [nq H][parts][D], stat fp64 [nq H][parts][3]: most of them cancels between the parts); parts: of a key tile's rows (part2 [parts][dk, dv][nk][KV][D])
    int32_t key_parts, parts, uneven;          // uneven: rows see unlike numbers of keys (the longest at least 1.5 times the mean)
    float *part, *stat, *part2;
    int32_t q_vec, k_vec, v_vec, do_vec, o32_vec;   // bytes per load that strides, base and width allow: 16, 8 or the element
    int32_t o_vec;                                 // results are stored four at a time
};

namespace sattn {

typedef __bf16 bf16;
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

// Fills tiles of ROWS rows (columns behind D: anything finite that the row holds - the other operand is 0 there, or the result is not
// stored).  Loads of 16 bytes go straight into LDS, 64 lanes an instruction, the swizzle applied to the source; nothing waits until landed().
// Where rows follow each other evenly, a thread's places in a tile are offsets that never change (off[]) on a base that moves from tile to tile:
// no address arithmetic per tile (it took a third of the plain forward's vector instructions).
template <typename T, int DP, int ROWS, int NT> struct Stage {
    using L = Tile<T, DP>;
    static constexpr int NC = ROWS * L::NCH, PER = (NC + NT - 1) / NT;
    static_assert(NC % 64 == 0, "whole waves");
    typedef __attribute__((address_space(3))) void *lp;
    typedef const __attribute__((address_space(1))) void *gp;
    uint32_t off[PER];
    // span(r): bytes from the tile's first row to row r
    template <typename Span> __device__ __forceinline__ void offsets(Span span, int D) {
        const int last = (D - 1) / Tr<T>::CH;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int s = min(i * NT + (int)threadIdx.x, NC - 1), r = s / L::NCH, c = (s % L::NCH) ^ L::swz(r);
            off[i] = span(r) + (uint32_t)min(c, last) * 16;
        }
    }
    // the rows from base on, all of them there
    __device__ __forceinline__ void even(u32x4 *tile, const T *base) const {
        const int w0 = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63);
        const char *p = reinterpret_cast<const char *>(base);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (NC % NT == 0 || i * NT + w0 < NC) __builtin_amdgcn_global_load_lds((gp)(p + off[i]), (lp)(tile + i * NT + w0), 16, 0, 0);
    }
    // any rows: row(r) points to row r
    template <typename Row> static __device__ __forceinline__ void any(u32x4 *tile, Row row, int D, int vec) {
        const int w0 = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63), last = (D - 1) / Tr<T>::CH;
#pragma unroll 1
        for (int i = 0; i < PER; ++i) {
            const int s = i * NT + (int)threadIdx.x, r = s / L::NCH, c = (s % L::NCH) ^ L::swz(r);
            if (NC % NT != 0 && i * NT + w0 >= NC) break;
            if (vec == 16) __builtin_amdgcn_global_load_lds((gp)(row(r) + min(c, last) * Tr<T>::CH), (lp)(tile + i * NT + w0), 16, 0, 0);
            else tile[s] = load_chunk<T>(row(r), c * Tr<T>::CH, D, vec);            // through registers: in LDS on return
        }
    }
};
// bytes of a tile of rows fit the offsets
__device__ __forceinline__ bool short_rows(int64_t stride, int rows, int size) { return stride >= 0 && stride * rows * size < (1ll << 31); }
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

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t cvt2(float a, float b) {                // one v_cvt_pk_bf16_f32
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// B operand of the second product from score-shaped registers; P and dS are rounded to the inputs' type here and nowhere else
__device__ __forceinline__ f32x4 pack_p(const f32x4 *p, float) { return p[0]; }
__device__ __forceinline__ bf16x8 pack_p(const f32x4 *p, bf16) {
    const u32x4 r = {cvt2(p[0][0], p[0][1]), cvt2(p[0][2], p[0][3]), cvt2(p[1][0], p[1][1]), cvt2(p[1][2], p[1][3])};
    return __builtin_bit_cast(bf16x8, r);
}
// what that rounding left over, rounded in turn: p to 16 bits through two products
__device__ __forceinline__ bf16x8 pack_rest(const f32x4 *p, bf16x8 hi) {
    const u32x4 h = __builtin_bit_cast(u32x4, hi);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = cvt2(p[i >> 1][(i & 1) * 2] - __uint_as_float(h[i] << 16), p[i >> 1][(i & 1) * 2 + 1] - __uint_as_float(h[i] & 0xffff0000u));
    return __builtin_bit_cast(bf16x8, r);
}
__device__ __forceinline__ f32x4 pack_rest(const f32x4 *, f32x4 hi) { return hi; }      // fp32 rounds nothing: never used

// tanh to a few ulp of fp32: near zero the odd rational [5/4] from the continued fraction x / (1 + x^2 / (3 + x^2 / (5 + ...))) (before rounding off by at most
// 4.7e-8, 6.2e-8 of tanh, for |x| <= 1; the products and the quotient round on top), else 1 - 2 / (1 + e^2x), which loses nothing there.
__device__ __forceinline__ float tanh_near(float x) {
    const float s = x * x;
    return x * (945.f + s * (105.f + s)) * rcp_(945.f + s * (420.f + s * 15.f));
}
__device__ __forceinline__ float tanh_(float x) {
    const float far = 1.f - 2.f * rcp_(1.f + exp2_(fabsf(x) * (2.f * LOG2E)));
    return fabsf(x) < 1.f ? tanh_near(x) : copysignf(far, x);
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
// over the four lane groups of one column: v_permlane16_swap of a register with itself puts its rows 0 and 2 (of 16 lanes) in one result and 1 and 3
// in the other, v_permlane32_swap its halves - vector instructions, where a shuffle goes through LDS
__device__ __forceinline__ float group_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float group_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// packed row -> (row, head within its group); 32-bit division where it does (a 64-bit one is over a hundred instructions)
__device__ __forceinline__ int row_of(int64_t r, int G) {
    if (G == 1) return (int)r;
    return r <= 0xffffffffll ? (int)((uint32_t)r / (uint32_t)G) : (int)(r / G);
}

// Row c of the wave (all four lane groups hold the same), as the kernels keep it per lane.
struct RowState {
    int row, head, lo, hi;
    float slope, pos[3];
};

__device__ __forceinline__ RowState row_state(const SceneAttnArgs &A, int kvh, int64_t r, int64_t R) {
    RowState s;
    const int64_t rr = r < R ? r : R - 1;
    s.row = row_of(rr, A.G);
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
// a value that all lanes share, in a scalar register
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

// Which tile a workgroup takes, heaviest first in rounds of one workgroup a CU, every other round backwards: a CU that got a heavy tile
// in one round gets a light one in the next.  (Causal masks: tiles differ by the length of the sequence.)  n: tiles, i: 0 .. n - 1, per: rounds' length.
__device__ __forceinline__ int snake(uint32_t i, uint32_t n, uint32_t per) {
    const uint32_t r = i / per, in = i - r * per, len = min(per, n - r * per);
    return (int)(r * per + (r & 1 ? len - 1 - in : in));
}
constexpr int CUS = 256;

// part i of n of the keys lo .. hi - 1, in whole tiles of BN
template <int BN> __device__ __forceinline__ void key_part(int &lo, int &hi, int i, int n) {
    const int64_t per = (int64_t)(((uint32_t)max(hi - lo, 0) + (uint32_t)(n * BN) - 1) / (uint32_t)(n * BN)) * BN, at = lo + per * i;
    lo = (int)min(at, (int64_t)hi);
    hi = (int)min(at + per, (int64_t)hi);
}

// Single values of a tile's N rows (N <= 64) straight into LDS: src is this lane's
template <int N> __device__ __forceinline__ void stage_values(float *dst, const void *src) {
    typedef __attribute__((address_space(3))) void *lp;
    typedef const __attribute__((address_space(1))) void *gp;
    if ((int)(threadIdx.x & 63) < N) __builtin_amdgcn_global_load_lds((gp)src, (lp)dst, 4, 0, 0);
}
// The coordinates of N keys from key on, one array an axis, axis a by wave a; last: the last key there is (it stands in for those behind it)
template <int AX, int N> __device__ __forceinline__ void stage_positions(float (*dst)[N], const SceneAttnArgs &A, const float *kpos, int key, int last) {
    const int a = uniform((int)(threadIdx.x >> 6));
    if (AX > 0 && a < A.axes) stage_values<N>(dst[a], kpos + (int64_t)min(key + (int)(threadIdx.x & 63), last) * A.axes + a);
}
// axes that the launch does not have
template <int AX, int N> __device__ __forceinline__ void clear_positions(float (*dst)[N], int axes) {
    if constexpr (AX > 0)
        for (int i = threadIdx.x; i < AX * N; i += 256)
            if (i / N >= axes) dst[i / N][i % N] = 0.f;
}
template <int AX, int N> __device__ __forceinline__ void read_positions(const float (*s)[N], int at, f32x4 &px, f32x4 &py, f32x4 &pz) {
    if constexpr (AX > 0) px = *reinterpret_cast<const f32x4 *>(&s[0][at]);
    if constexpr (AX > 1) {
        py = *reinterpret_cast<const f32x4 *>(&s[1][at]);
        pz = *reinterpret_cast<const f32x4 *>(&s[2][at]);
    }
}

// Scores in base 2 from raw products, the constants of one launch folded together.  CAP and AX (0, 1, or 3 for two and three
// coordinates) are compiled in: the kernels are bound by vector instructions per score, not by the products.
// Capped: with s = raw^2 the rational tanh_near() and both factors become raw (k + s (n1 + s n2)) / (1 + s (d1 + s d2)), eight instructions.
// Scores of a trained model lie well inside the cap, so a wave seldom takes the form for |raw| >= edge.
// FINE (fp32): quotient and root to half an ulp - a score of 30 off by one more ulp is 2e-6 in its probability.
template <bool CAP, int AX, bool FINE> struct Score {
    float k, arg, cap2, inv2, edge, n1, n2, d1, d2;
    __device__ __forceinline__ Score(const SceneAttnArgs &A) : k(uniform(A.scale * LOG2E)) {
        if constexpr (CAP) {
            arg = uniform(A.scale / A.cap);
            cap2 = uniform(A.cap * LOG2E);
            inv2 = uniform(1.f / cap2);
            edge = uniform(fabsf(arg) > 1e-8f && fabsf(arg) < 1e8f ? 1.f / fabsf(arg) : 0.f);      // else arg^4 leaves fp32's range
            const float a2 = arg * arg;
            n1 = uniform(k * a2 * (105.f / 945.f));
            n2 = uniform(k * a2 * a2 * (1.f / 945.f));
            d1 = uniform(a2 * (420.f / 945.f));
            d2 = uniform(a2 * a2 * (15.f / 945.f));
        }
    }
    // N vectors of raw products to scores without the distance
    template <int N> __device__ __forceinline__ void apply(f32x4 *x) const {
        if constexpr (!CAP) {
#pragma unroll
            for (int n = 0; n < N; ++n) x[n] *= k;
            return;
        }
        bool far = false;
#pragma unroll
        for (int n = 0; n < N; ++n) far = far || !(fmaxf(fmaxf(fabsf(x[n][0]), fabsf(x[n][1])), fmaxf(fabsf(x[n][2]), fabsf(x[n][3]))) < edge);
        if (__any(far)) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[n][i] = cap2 * tanh_(x[n][i] * arg);
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float s = x[n][i] * x[n][i];
                    const float num = x[n][i] * fmaf(s, fmaf(s, n2, n1), k), den = fmaf(s, fmaf(s, d2, d1), 1.f), r = rcp_(den);
                    x[n][i] = num * r;
                    if constexpr (FINE) x[n][i] = fmaf(fmaf(-den, x[n][i], num), r, x[n][i]);
                }
        }
    }
    // 1 - tanh^2 from such a score
    __device__ __forceinline__ f32x4 slope_of(f32x4 x) const {
        const f32x4 t = x * inv2;
        return 1.f - t * t;
    }
    static __device__ __forceinline__ float dist(float x, float y, float z) {
        if constexpr (AX == 1) return fabsf(x);
        const float q = x * x + y * y + z * z;
        float r = __builtin_amdgcn_sqrtf(q);
        if constexpr (FINE) r = q > 0.f && q < __builtin_inff() ? fmaf(fmaf(-r, r, q), 0.5f * rcp_(r), r) : r;
        return r;
    }
    // of one row's position to four positions
    static __device__ __forceinline__ f32x4 dist4(const float *a, f32x4 px, f32x4 py, f32x4 pz) {
        f32x4 d;
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = AX == 1 ? fabsf(a[0] - px[i]) : dist(a[0] - px[i], a[1] - py[i], a[2] - pz[i]);
        return d;
    }
};

// Without cap and distance the kernels mask raw products with -inf and apply the factor later.  -inf times 0 is NaN, so a scale that is 0 (or a
// denormal, which a product may flush) takes the form that applies the factor first: one axis of no length.
inline bool factor_last(const SceneAttnArgs &A) { return A.axes == 0 && __builtin_fabsf(A.scale) >= 0x1p-126f; }

// the same with everything read at run time (the slow forms)
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
                const u32x2 h = {cvt2(v[0], v[1]), cvt2(v[2], v[3])};
                *reinterpret_cast<u32x2 *>(p + d) = h;
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (d + i < D) p[d + i] = (T)v[i];
}

}  // namespace sattn
