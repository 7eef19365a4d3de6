// Device code of libtoa_muon.so: see include/toa_muon.h for what the operators compute.
//
// Every matrix is worked on in its wide orientation (s rows, w columns, s <= w; a tall one is
// read and written turned).  Per step k of the series, with X = X_k, completing the square:
//     S = X X^T + h I,               h = b / 2c          (symmetric: lower tiles only, mirrored)
//     P = c S S + (a - b h / 2) I                        (symmetric too)
//     X' = P X                       = a X + b (X X^T) X + c (X X^T)^2 X
// and for the gradient, with the cotangent Y of X':
//     M = Y X^T + X Y^T,   N = c (M S + S M),   Y_prev = P Y + N X.
// All of them are sums of products A B^T of row-major operands, so ONE kernel computes them: a
// tile of up to two products with a common sum, plus a multiple of the unit matrix, stored in both
// orientations (X and X^T; for the symmetric ones the mirror image).  No stage reads a third
// matrix; measured, the read of one at a tile's end cost as much as 15 % of its products.
// (Where c is zero, or c h^2 large beside a: S = X X^T, P = c S S + b S + a I,
// N = c (M S + S M) + b M, with that third matrix.)
//
// Two steps at once, where X is wide: the S of the next step is P S P, so X itself is needed once:
//     S = X X^T,  P = c S S + b S + a I,  T = P S,  S' = T P + h I,  P' = c S' S' + (a - b h / 2) I,
//     Q = P' P,   X'' = Q X
// takes 3 w + 5 s instead of 6 w + 2 s (times s^2).  It is no less accurate than two single steps as
// long as the first S is kept without h: there X X^T is small beside h I, whose rounding would pass
// through T.  (Three at once lose: P S P magnifies the error of S by a^2.)
//
// Operands.  The matrix cores multiply halves; an operand element is kept as hi + lo, two halves
// that together carry 22 bits, and a product is hi hi + hi lo + lo hi with float32 sums (what is
// dropped, lo lo, is 2^-24 of it on average; small_kernel, whose sums are too short to hide that, has
// it in float32).  Halves have few exponents, so every matrix is stored times a power of two that takes its bound to 2^13..2^14: |X_k| <= max of the polynomial on the previous
// interval (from the start's norm, 1 or less), and products of such bounds for the others.  An
// element is at most the spectral norm, so nothing overflows, and what lies 2^-15 below the bound
// still has all its bits.  ("half" operands keep hi alone: 11 bits, in the last step of bfloat16 calls
// whose series magnifies their rounding little.)
//
// Layout.  An operand lies the way the matrix instructions read it: by blocks of 32 rows, and in
// them by pieces of 4 KiB, [32 hi | 32 lo] of 32 columns or 64 halves of 64 columns of each row.  A
// piece is eight chunks of eight columns, 16 bytes of every row, rows next to each other: two chunks
// are the 1 KiB that the lanes of a wave hold for one instruction.  Columns beyond the matrix are
// zero up to a multiple of 64; rows beyond it, up to a multiple of 32, hold anything.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace toa_muon {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMaxGroups = 16;   // distinct shapes in one launch
constexpr int kMaxSteps = 32;
constexpr int kMaxParts = 256;   // partial sums per matrix
constexpr int kBlock = 128;      // elements of an 8-bit block
constexpr int kPiece = 128;      // bytes of a row that one tile step consumes
constexpr int kRows = 32;        // rows of a block of an operand
constexpr int kPad = 64;         // columns are padded to a multiple of this

// What a kernel needs to know of the caller's tensors, in the wide orientation.
struct MatRec {
    const void *g;     // the matrix (orthogonalize), or its gradient (step)
    const void *aux;   // the momentum (step), or the cotangent (gradient)
    void *out;
    float *scales;     // of an 8-bit momentum
    int64_t g_rs, g_cs, aux_rs, aux_cs, out_rs, out_cs;
    float rate, keep;  // out <- keep * out - rate * result (step), or rate * result
    int s, w;
};

// Sums over a matrix and what follows from them.
struct MatNorm {
    double x_scale;    // 2^e / (|G| + eps): what G is multiplied with on its way to X_0
    double y_scale;    // 2^e for the cotangent
    double size;       // |G|_F
    double plus;       // |G|_F + eps
    double y_size;     // |Y|_F of the cotangent that was measured last,
    int y_step, y_exp; // of which iterate it is, and the power of two it is stored with
};

struct Group {         // matrices of one shape
    int64_t base;      // bytes from the workspace to the first one's region
    int64_t stride;    // bytes from one region to the next
    int64_t kept_base, kept_stride;  // the same in the buffer of kept iterates
    int s, w, mat0;
    int tile0, tiles, all;  // workgroups of this launch: first, per matrix, of all its matrices
};

struct Shapes {
    int n;
    Group g[kMaxGroups];
};

// Where a matrix's buffers lie: at an offset into its region of the workspace or, with this bit set, of
// the buffer that keeps the iterates between the forward pass and the gradient.
constexpr int64_t kKept = (int64_t)1 << 62;

struct Region {
    char *own, *kept;
    __device__ Region(char *ws, char *kept_, const Group &g, int mat)
        : own(ws + g.base + mat * g.stride), kept(kept_ + g.kept_base + mat * g.kept_stride) {}
    __device__ char *operator+(int64_t offset) const {
        return offset & kKept ? kept + (offset & ~kKept) : own + offset;
    }
};

// The caller's tensors come as addresses in records: without this they would be read and written
// with instructions that look for LDS behind every address.
#define TOA_GLOBAL __attribute__((address_space(1)))
template <typename T> __device__ inline const TOA_GLOBAL T *global(const void *p) {
    return (const TOA_GLOBAL T *)p;
}
template <typename T> __device__ inline TOA_GLOBAL T *global(void *p) { return (TOA_GLOBAL T *)p; }

__device__ inline float toFloat(float v) { return v; }
__device__ inline float toFloat(_Float16 v) { return (float)v; }
__device__ inline float toFloat(__bf16 v) { return (float)v; }
template <typename T> __device__ inline T fromFloat(float v) { return (T)v; }

// The group and the matrix a workgroup belongs to; `tile` becomes the tile's number in it.
__device__ inline int findGroup(const Shapes &sh, int &tile, int &mat) {
    int k = 0;
    while (k + 1 < sh.n && tile >= sh.g[k + 1].tile0) ++k;
    tile -= sh.g[k].tile0;
    mat = tile / sh.g[k].tiles;
    tile -= mat * sh.g[k].tiles;
    return k;
}

__device__ inline double blockSum(double v, double *lds) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (unsigned i = 0; i < blockDim.x / 64; ++i) s += lds[i];
    __syncthreads();
    return s;
}

// ---- the records -----------------------------------------------------------------------------

constexpr int kFill = 32;
struct FillArgs {
    MatRec r[kFill];
};
// Records travel in the launch's own arguments: no host buffer has to outlive the call, and a
// captured graph holds them by value.  Few of them come with the first pass over the matrices, which
// leaves them in the workspace for the others, and that batch's factors are made by the pass that
// makes its operands: two launches less, 5 us of 195 for one 1024^2 matrix.
constexpr int kFew = 24;
__global__ void fill_kernel(FillArgs a, MatRec *dst, int n) {
    const int i = threadIdx.x;
    if (i < n) dst[i] = a.r[i];
}

// A copy in scalar registers.
__device__ inline MatRec uniform(const MatRec *p) {
    MatRec r;
    constexpr int kWords = sizeof(MatRec) / 4;
    int words[kWords];
    __builtin_memcpy(words, p, sizeof(MatRec));
#pragma unroll
    for (int i = 0; i < kWords; ++i) words[i] = __builtin_amdgcn_readfirstlane(words[i]);
    __builtin_memcpy(&r, words, sizeof(MatRec));
    return r;
}

// ---- the momentum and the norms --------------------------------------------------------------
//
// One pass over G (or g and M), in memory order where the matrix is dense: sums of squares in
// double (no overflow, no dependence on how many there are), a partial sum per workgroup, added
// up in a fixed order by factors_kernel.  The look-ahead U is formed in 32 bits, here and where it is
// made an operand: its own rounding (2^-24) is far below the operands' (2^-22).
//
// Bound by HBM: GPT-2-medium's 302 million elements in bfloat16, 6 bytes each, 318 us = 5.7 TB/s (a
// large copy reaches 5.1).  With 8-bit blocks, 4 bytes an element, by the arithmetic in double: 75.5
// million in 134 us = 2.3 TB/s.

enum { kSumG = 0, kSumAux = 1, kMomentum = 2, kMomentumF32 = 3, kMomentumI8 = 4 };

struct StepArgs {      // what the momentum's update needs
    double momentum;
    float sign;
    int nesterov;
};

struct SumArgs {
    Shapes sh;
    const MatRec *recs;
    double *parts;     // [matrix][kMaxParts]
    StepArgs step;
    int64_t per[kMaxGroups];  // elements per workgroup, a multiple of 2048
    int few;                  // so many records are here, and `recs` is where they go
    MatRec r[kFew];
};
static_assert(sizeof(SumArgs) <= 4096, "a launch's arguments");

template <typename T> __device__ inline void load8(const T *p, int valid, float (&v)[8]) {
    if (valid >= 8 && ((uintptr_t)p & 15) == 0) {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
        for (unsigned q = 0; q < 8 / (16 / sizeof(T)); ++q) {
            const vec t = global<vec>(p)[q];
#pragma unroll
            for (unsigned i = 0; i < 16 / sizeof(T); ++i) v[q * (16 / sizeof(T)) + i] = toFloat((T)t[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < valid ? toFloat(global<T>(p)[i]) : 0.f;
    }
}

template <typename T> __device__ inline void store8(T *p, int valid, const float (&v)[8]) {
    if (valid >= 8 && ((uintptr_t)p & 15) == 0) {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
        for (unsigned q = 0; q < 8 / (16 / sizeof(T)); ++q) {
            vec t;
#pragma unroll
            for (unsigned i = 0; i < 16 / sizeof(T); ++i) t[i] = fromFloat<T>(v[q * (16 / sizeof(T)) + i]);
            global<vec>(p)[q] = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) global<T>(p)[i] = fromFloat<T>(v[i]);
    }
}

// Largest magnitude of the 16 lanes that share an 8-bit block, as bits (a NaN is the largest).
__device__ inline unsigned long long blockPeak(unsigned long long m) {
#pragma unroll
    for (int o = 8; o; o >>= 1) {
        const unsigned long long t = __shfl_xor(m, o);
        m = t > m ? t : m;
    }
    return m;
}

// The scale of a block whose largest magnitude has the bits `peak`: NaN where that is not finite,
// so that the whole block stands for NaN.
__device__ inline float scaleOf(unsigned long long peak) {
    if (peak >= 0x7ff0000000000000ull) return __int_as_float(0x7fc00000);
    return (float)(__longlong_as_double((long long)peak) / 127.0);
}

// v / scale rounded half to even: the multiple that v times the reciprocal suggests and, where that
// lies next to a border, its exact remainder decides.
__device__ inline int codeOf(double v, float scale, double reciprocal) {
    if (!(scale > 0.f)) return 0;
    const double t = v * reciprocal;
    double q = __builtin_rint(t);
    if (__builtin_fabs(t - q) > 0.499999) {
        const double rest = __builtin_fma(-q, (double)scale, v), half = 0.5 * (double)scale;
        const bool odd = ((int)q & 1) != 0;
        if (rest > half || (rest == half && odd)) q += 1.0;
        if (rest < -half || (rest == -half && odd)) q -= 1.0;
    }
    // (a scale too small for float32's normal range may be rounded to half of peak / 127)
    const int code = (int)q;
    return code > 127 ? 127 : code < -127 ? -127 : code;
}

__device__ inline void unpack8(int64_t v, int8_t (&c)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = (int8_t)(v >> (8 * i));
}

__device__ inline int64_t pack8(const int8_t (&c)[8]) {
    uint64_t v = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v |= (uint64_t)(uint8_t)c[i] << (8 * i);
    return (int64_t)v;
}

// A thread's share of the elements from `from` (a multiple of 128) to `to`: updates the momentum
// there and returns the sum of squares.
template <typename T, int KIND>
__device__ double sumPass(const MatRec &r, const StepArgs &a, int64_t from, int64_t to) {
    const T *src = (const T *)(KIND == kSumAux ? r.aux : r.g);
    const int64_t rs = KIND == kSumAux ? r.aux_rs : r.g_rs;
    const int64_t cs = KIND == kSumAux ? r.aux_cs : r.g_cs;
    // the steps' tensors are dense by contract
    const bool flat = KIND >= kMomentum || (cs == 1 && rs == r.w) || (rs == 1 && cs == r.s);
    double sum = 0.0;
    // In double: values next to a border (decay rates are short decimals, 16-bit values short
    // binary fractions, so ties are common) round as the exact sum does, whatever the type.
    auto next = [&](double m, float grad) { return a.momentum * m + (double)grad; };
    for (int64_t e = from + (int64_t)threadIdx.x * 8; (e & ~(int64_t)127) < to; e += (int64_t)blockDim.x * 8) {
        // (the bound keeps the 16 lanes of an 8-bit block together)
        const int valid = e >= to ? 0 : to - e < 8 ? (int)(to - e) : 8;
        float v[8];
        if (KIND == kSumG || KIND == kSumAux) {
            if (flat) {
                load8(src + e, valid, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t x = e + i, row = x / r.w, col = x - row * r.w;
                    v[i] = i < valid ? toFloat(global<T>(src)[row * rs + col * cs]) : 0.f;
                }
            }
        } else {
            float grad[8], m[8];
            load8(src + e, valid, grad);
#pragma unroll
            for (int i = 0; i < 8; ++i) grad[i] *= a.sign;
            if (KIND == kMomentumI8) {
                int8_t *codes = (int8_t *)const_cast<void *>(r.aux) + e;
                const float old = valid ? global<float>(r.scales)[e >> 7] : 0.f;
                double d[8];
                unsigned long long peak = 0;
                int8_t c[8];
                if (valid == 8 && ((uintptr_t)codes & 7) == 0) {
                    unpack8(*global<int64_t>(codes), c);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) c[i] = i < valid ? global<int8_t>(codes)[i] : (int8_t)0;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    d[i] = i < valid ? next((double)c[i] * (double)old, grad[i]) : 0.0;
                    const unsigned long long mag =
                        (unsigned long long)__double_as_longlong(d[i]) & 0x7fffffffffffffffull;
                    peak = mag > peak ? mag : peak;
                }
                const float scale = scaleOf(blockPeak(peak));
                const double reciprocal = 1.0 / (double)scale;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    c[i] = (int8_t)codeOf(d[i], scale, reciprocal);
                    m[i] = (float)c[i] * scale;
                }
                if (valid == 8 && ((uintptr_t)codes & 7) == 0) {
                    *global<int64_t>((void *)codes) = pack8(c);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < valid) global<int8_t>((void *)codes)[i] = c[i];
                }
                if (valid && (e & 127) == 0) global<float>((void *)r.scales)[e >> 7] = scale;
            } else if (KIND == kMomentumF32) {
                float *buf = (float *)const_cast<void *>(r.aux) + e;
                load8(buf, valid, m);
#pragma unroll
                for (int i = 0; i < 8; ++i) m[i] = (float)next(m[i], grad[i]);
                store8(buf, valid, m);
            } else {
                T *buf = (T *)const_cast<void *>(r.aux) + e;
                load8(buf, valid, m);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    m[i] = toFloat(fromFloat<T>((float)next(m[i], grad[i])));
                store8(buf, valid, m);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = a.nesterov ? __builtin_fmaf((float)a.momentum, m[i], grad[i]) : m[i];
                if (i >= valid) v[i] = 0.f;  // (0 * NaN of a block that stands for NaN)
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fma((double)v[i], (double)v[i], sum);
    }
    return sum;
}

template <typename T, int KIND>
__global__ __launch_bounds__(256) void sum_kernel(SumArgs a) {
    __shared__ double lds[4];
    int part = blockIdx.x, mat;
    const int gi = findGroup(a.sh, part, mat);
    mat += a.sh.g[gi].mat0;
    if (a.few && blockIdx.x == 0)
        for (int i = threadIdx.x; i < a.few * (int)(sizeof(MatRec) / 4); i += 256)
            ((int *)const_cast<MatRec *>(a.recs))[i] = ((const int *)a.r)[i];
    const MatRec r = uniform(a.few ? a.r + mat : a.recs + mat);
    const int64_t n = (int64_t)r.s * r.w, from = part * a.per[gi];
    const int64_t to = from + a.per[gi] < n ? from + a.per[gi] : n;
    const double sum = blockSum(sumPass<T, KIND>(r, a.step, from, to), lds);
    if (threadIdx.x == 0) a.parts[(int64_t)mat * kMaxParts + part] = sum;
}

// ---- scales and factors ----------------------------------------------------------------------

struct Factor {
    float acc, add, turn, diag;  // result = acc * sum + add * E + diag * I;
                                 // turn: the sum is multiplied with it between the products
};

struct Series {
    int steps, square;              // square: S carries h
    int paired;                     // so many steps are taken by twos
    int halves;                     // bfloat16: the last step's operands may carry 11 bits
    float a, b, c;
    double eps, h, unit;            // unit: the multiple of I in P
    double x[kMaxSteps + 1];        // bound of |X_k| from a start of norm 1
    double r[kMaxSteps];            // bound of |p(t) / t| on [0, x_k], which is |P|'s
    double d[kMaxSteps];            // bound of |p'| on [0, x_k]
};

struct FactorArgs {
    Series q;
    const double *parts, *parts_y;  // parts_y: of the cotangent, or null
    MatNorm *norms;
    Factor *factors;                // [matrix][stages]
    int stages;
    int nparts[kMaxGroups], mat_end[kMaxGroups], ngroups;
    int measured;                   // parts_y are of this iterate's cotangent as it is stored, or -1
};

// The power of two that takes a bound to at most 2^14.
__device__ inline int expOf(double bound) {
    if (!(bound > 1e-36)) bound = 1e-36;
    const int e = 13 - ilogb(bound);
    return e > 120 ? 120 : e < -110 ? -110 : e;
}

__device__ inline double startOf(double size, double eps) {
    const double s0 = size / (size + eps);
    return s0 > 1e-30 && s0 <= 1.0 ? s0 : s0 <= 1e-30 ? 1e-30 : 1.0;  // NaN: as if 1
}

// The arrays of a series, read by thread number: in LDS.
struct SeriesTable {
    double x[kMaxSteps + 1], r[kMaxSteps], d[kMaxSteps];
    __device__ void load(const Series &q) {  // by all threads; a barrier has to follow
        const int i = threadIdx.x;
        if (i <= q.steps) x[i] = q.x[i];
        if (i < q.steps) {
            r[i] = q.r[i];
            d[i] = q.d[i];
        }
    }
};

// Bounds of one matrix's iterates and cotangents.
struct Bounds {
    const Series &q;
    const SeriesTable &table;
    const double start;
    double ysize;       // of the cotangent of X_ystep, which is stored times 2^yexp
    int ystep, yexp_;
    __device__ Bounds(const Series &q_, const SeriesTable &table_, double size, double ysize_)
        : q(q_), table(table_), start(startOf(size, q_.eps)),
          ysize(ysize_ == ysize_ && ysize_ < 1e300 ? ysize_ : 1.0), ystep(q_.steps),
          yexp_(expOf(ysize)) {}
    __device__ double x(int i) const {  // of X_i
        double grown = start;
        for (int j = 0; j < i; ++j) grown *= table.r[j];
        return grown < table.x[i] ? grown : table.x[i];
    }
    __device__ double y(int i) const {  // of the cotangent of X_i
        double v = ysize;
        for (int j = ystep - 1; j >= i; --j) v *= table.d[j];
        return v;
    }
    __device__ int yexp(int i) const { return i == ystep ? yexp_ : expOf(y(i)); }
};

__device__ inline MatNorm normOf(const Bounds &b, double size) {
    const double plus = size + b.q.eps;
    return {ldexp(1.0 / plus, expOf(b.x(0))), ldexp(1.0, b.yexp_), size, plus, b.ysize, b.ystep, b.yexp_};
}

// Factors of a step: 4 of its own, so 8 of a pair's; in the gradient 3 more, behind all of those.
constexpr int kStepFactors = 4;

// The factors of the stages of steps t and t + 1 taken at once: f[0..6] for S, P, T, S', P', Q, X''.
__device__ inline void pairFactors(const Bounds &b, int t, Factor *f) {
    const Series &q = b.q;
    const double x = b.x(t), x2 = x * x, x1 = b.x(t + 1), r = b.table.r[t], r1 = b.table.r[t + 1];
    const int ex = expOf(x), es = expOf(x2), ep = expOf(r), et = expOf(r * x2), eq = expOf(r * r1);
    const int es1 = expOf(q.square ? fmax(fabs(q.h), fabs(q.h + x1 * x1)) : x1 * x1), ep1 = expOf(r1);
    const int ex2 = t + 2 == q.steps ? 0 : expOf(b.x(t + 2));
    f[0] = {ldexpf(1.f, es - 2 * ex), 0.f, 1.f, 0.f};
    f[1] = {ldexpf(q.c, ep - 2 * es), ldexpf(q.b, ep - es), 1.f, ldexpf(q.a, ep)};
    f[2] = {ldexpf(1.f, et - ep - es), 0.f, 1.f, 0.f};
    f[3] = {ldexpf(1.f, es1 - et - ep), 0.f, 1.f, (float)(q.square ? ldexp(q.h, es1) : 0.0)};
    f[4] = {ldexpf(q.c, ep1 - 2 * es1), q.square ? 0.f : ldexpf(q.b, ep1 - es1), 1.f,
            (float)ldexp(q.unit, ep1)};
    f[5] = {ldexpf(1.f, eq - ep1 - ep), 0.f, 1.f, 0.f};
    f[6] = {ldexpf(1.f, ex2 - eq - ex), 0.f, 1.f, 0.f};
}

// The factors of step t's stages: f[0..2] for S, P, X'; back[0..2] (or null) for M, N, Y.
__device__ inline void stepFactors(const Bounds &b, int t, Factor *f, Factor *back) {
    const Series &q = b.q;
    const double x = b.x(t), x2 = x * x, ab = fabs((double)q.b), ac = fabs((double)q.c);
    const double sbound = q.square ? fmax(fabs(q.h), fabs(q.h + x2)) : x2;
    const int ex = expOf(x), es = expOf(sbound), ep = expOf(b.table.r[t]);
    const bool last = t + 1 == q.steps;
    const int ex1 = last && !back ? 0 : expOf(b.x(t + 1));
    const float add = q.square ? 0.f : q.b;
    f[0] = {ldexpf(1.f, es - 2 * ex), 0.f, 1.f, (float)(q.square ? ldexp(q.h, es) : 0.0)};
    f[1] = {ldexpf(q.c, ep - 2 * es), ldexpf(add, ep - es), 1.f, (float)ldexp(q.unit, ep)};
    f[2] = {ldexpf(1.f, ex1 - ep - ex), 0.f, 1.f, 0.f};
    if (!back) return;
    const double y1 = b.y(t + 1);
    const int ey1 = b.yexp(t + 1), ey = t ? b.yexp(t) : 0;
    // (where N X is nothing beside P Y, N needs no more range than to be added to it)
    const int em = expOf(2.0 * x * y1);
    const int en = min(expOf((ab + 2.0 * ac * x2) * 2.0 * x * y1), ep + ey1 - ex + 24);
    back[0] = {ldexpf(1.f, em - ey1 - ex), 0.f, 1.f, 0.f};
    back[1] = {ldexpf(q.c, en - em - es), ldexpf(add, en - em), 1.f, 0.f};
    back[2] = {ldexpf(1.f, ey - en - ex), 0.f, ldexpf(1.f, (en + ex) - (ep + ey1)), 0.f};
}

// By a whole workgroup: a matrix's norms and, if it is the one to `write`, those and the factors of all
// stages into the workspace, a thread for each step.
__device__ inline MatNorm makeFactors(const FactorArgs &a, int mat, int np, bool write,
                                      SeriesTable &table, double *lds) {
    const int t = threadIdx.x;
    table.load(a.q);
    const double ysize =
        a.parts_y ? sqrt(blockSum(t < np ? a.parts_y[(int64_t)mat * kMaxParts + t] : 0.0, lds)) : 0.0;
    const double size = sqrt(blockSum(t < np ? a.parts[(int64_t)mat * kMaxParts + t] : 0.0, lds));
    const Bounds b(a.q, table, size, ysize);
    const MatNorm norm = normOf(b, size);
    if (!write) return norm;
    if (t == 0) a.norms[mat] = norm;
    Factor *f = a.factors + (int64_t)mat * a.stages + kStepFactors * t;
    if (t < a.q.steps) {
        if (t >= a.q.paired)
            stepFactors(b, t, f,
                        a.parts_y ? a.factors + (int64_t)mat * a.stages + kStepFactors * a.q.steps + 3 * t
                                  : nullptr);
        else if (t % 2 == 0)
            pairFactors(b, t, f);
    }
    return norm;
}

// One workgroup per matrix.
__global__ __launch_bounds__(256) void factors_kernel(FactorArgs a) {
    __shared__ double lds[4];
    __shared__ SeriesTable table;
    const int mat = blockIdx.x, t = threadIdx.x;
    int k = 0;
    while (k + 1 < a.ngroups && mat >= a.mat_end[k]) ++k;
    const int np = a.nparts[k];
    if (a.measured < 0) {
        makeFactors(a, mat, np, true, table, lds);
        return;
    }
    // on the way back: bounds of the cotangents from this one on follow its norm
    table.load(a.q);
    const double stored = sqrt(blockSum(t < np ? a.parts_y[(int64_t)mat * kMaxParts + t] : 0.0, lds));
    const MatNorm n = a.norms[mat];
    Bounds b(a.q, table, n.size, n.y_size);
    b.ystep = n.y_step;
    b.yexp_ = n.y_exp;
    const double bound = b.y(a.measured);
    b.yexp_ = b.yexp(a.measured);
    b.ystep = a.measured;
    const double now = ldexp(stored, -b.yexp_);
    b.ysize = now > 0.0 && now < bound ? now : bound;  // (nothing, or NaN: as before)
    __syncthreads();  // (everybody has read the norms)
    if (t == 0) a.norms[mat] = normOf(b, n.size);
    if (t < a.measured)
        stepFactors(b, t, a.factors + (int64_t)mat * a.stages + kStepFactors * t,
                    a.factors + (int64_t)mat * a.stages + kStepFactors * a.q.steps + 3 * t);
}

// ---- operands ----------------------------------------------------------------------------------

// Where eight consecutive columns, from a multiple of 8 on, of a row of an operand lie; `ld` is the
// bytes of a row.  Their low halves follow 2 KiB behind.
__device__ inline char *chunkOf(char *operand, int64_t ld, int row, int col, bool split) {
    const int piece = split ? col >> 5 : col >> 6, chunk = split ? (col >> 3) & 3 : (col >> 3) & 7;
    return operand + (int64_t)(row / kRows) * kRows * ld + (int64_t)piece * kRows * kPiece +
           chunk * 512 + row % kRows * 16;
}

__device__ inline void storeOperand(char *to, const float (&v)[8], bool split) {
    half8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi[i] = (_Float16)v[i];
        lo[i] = (_Float16)(v[i] - (float)hi[i]);
    }
    *global<half8>(to) = hi;
    if (split) *global<half8>(to + 2048) = lo;
}

__device__ inline void loadOperand(const char *from, float (&v)[8]) {  // 22-bit operands only
    const half8 hi = *global<half8>(from), lo = *global<half8>(from + 2048);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)hi[i] + (float)lo[i];
}

// Bytes of an operand row of `cols` padded columns.
__host__ __device__ inline int64_t rowBytes(int64_t padded, bool split) {
    return padded * (split ? 4 : 2);
}

__host__ __device__ inline int64_t padded(int64_t n) { return (n + kPad - 1) / kPad * kPad; }

enum { kPackG = 0, kPackAux = 1, kPackM = 2, kPackMF32 = 3, kPackMI8 = 4 };

struct PackArgs {
    Shapes sh;
    const MatRec *recs;
    const MatNorm *norms;
    char *ws, *kept;
    int64_t off[kMaxGroups], off_t[kMaxGroups];  // of the operand and of its transpose
    StepArgs step;
    int split;
    FactorArgs f;  // FEW: what is to be made of the sums on the way
};
static_assert(sizeof(PackArgs) <= 4096, "a launch's arguments");

// An element of G, of the step's U, or of the cotangent, `at` elements behind the first.
template <typename T, int KIND>
__device__ inline float element(const MatRec &r, const StepArgs &a, int64_t at) {
    float v = toFloat(global<T>(KIND == kPackAux ? r.aux : r.g)[at]);
    if (KIND >= kPackM) {
        float m;
        if (KIND == kPackMI8)
            m = (float)global<int8_t>(r.aux)[at] * global<float>(r.scales)[at >> 7];
        else if (KIND == kPackMF32)
            m = global<float>(r.aux)[at];
        else
            m = toFloat(global<T>(r.aux)[at]);
        v = a.nesterov ? __builtin_fmaf((float)a.momentum, m, a.sign * v) : m;
    }
    return v;
}

// Eight elements of G (U, the cotangent), consecutive in memory from `at` on.
template <typename T, int KIND>
__device__ inline void elements8(const MatRec &r, const StepArgs &a, int64_t at, int valid, float (&v)[8]) {
    load8((const T *)(KIND == kPackAux ? r.aux : r.g) + at, valid, v);
    if (KIND < kPackM) return;
    float m[8];
    if (KIND == kPackMI8) {
        const int8_t *p = (const int8_t *)r.aux + at;
        int8_t c[8];
        if (valid >= 8 && ((uintptr_t)p & 7) == 0) {
            unpack8(*global<int64_t>(p), c);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = i < valid ? global<int8_t>(p)[i] : (int8_t)0;
        }
        // (they lie in one block, or in two)
        const int64_t last = at + (valid < 8 ? valid : 8) - 1;
        const float s0 = global<float>(r.scales)[at >> 7], s1 = global<float>(r.scales)[last >> 7];
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = (float)c[i] * ((at + i) >> 7 == at >> 7 ? s0 : s1);
    } else if (KIND == kPackMF32) {
        load8((const float *)r.aux + at, valid, m);
    } else {
        load8((const T *)r.aux + at, valid, m);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = a.nesterov ? __builtin_fmaf((float)a.momentum, m[i], a.sign * v[i]) : m[i];
}

// G (or the step's U, or the cotangent) -> the operand and its transpose, by tiles of 64 x 64.  Eight
// elements that are neighbours in memory are eight columns of one of the two and go there at once;
// the other is made through LDS.  HBM-bound: 4 bytes (bfloat16 and its momentum) in, 8 out, GPT-2-medium's
// 302 million elements in 676 us = 5.4 TB/s.
template <typename T, int KIND, bool FEW>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a) {
    __shared__ float tile[64][65];  // [operand row or column][the other]
    __shared__ SeriesTable table;
    __shared__ double lds[4];
    int t = blockIdx.x, mat;
    const int gi = findGroup(a.sh, t, mat);
    const Group &g = a.sh.g[gi];
    const Region region(a.ws, a.kept, g, mat);
    mat += g.mat0;
    const MatRec &r = a.recs[mat];
    const int across = (int)(padded(g.w) / 64);
    const int i0 = t / across * 64, j0 = t % across * 64;
    const MatNorm norm =
        FEW ? makeFactors(a.f, mat, a.f.nparts[gi], t == 0, table, lds) : a.norms[mat];
    const double scale = KIND == kPackAux ? norm.y_scale : norm.x_scale;
    const int64_t rs = KIND == kPackAux ? r.aux_rs : r.g_rs, cs = KIND == kPackAux ? r.aux_cs : r.g_cs;
    // "lines" run along the smaller stride: rows of the operand, or (turned) its columns
    const bool by_rows = cs <= rs;
    const int64_t along = by_rows ? cs : rs, across_lines = by_rows ? rs : cs;
    const int lines = by_rows ? g.s : g.w, length = by_rows ? g.w : g.s;
    const int line0 = by_rows ? i0 : j0, at0 = by_rows ? j0 : i0;
    const int64_t ld = rowBytes(padded(g.w), a.split), ld_t = rowBytes(padded(g.s), a.split);
    char *const direct = region + (by_rows ? a.off[gi] : a.off_t[gi]);
    char *const turned = region + (by_rows ? a.off_t[gi] : a.off[gi]);
    const int64_t direct_ld = by_rows ? ld : ld_t, turned_ld = by_rows ? ld_t : ld;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int q = half * 256 + threadIdx.x, d = q >> 3, c = (q & 7) * 8;
        const int line = line0 + d, valid = line < lines ? length - at0 - c : 0;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
        if (valid > 0) {
            const int64_t at = line * across_lines + (at0 + c) * along;
            if (along == 1) {
                elements8<T, KIND>(r, a.step, at, valid, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < valid) v[i] = element<T, KIND>(r, a.step, at + i * along);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < valid ? (float)((double)v[i] * scale) : 0.f;
        }
        if (line < lines) storeOperand(chunkOf(direct, direct_ld, line, at0 + c, a.split), v, a.split);
#pragma unroll
        for (int i = 0; i < 8; ++i) tile[d][c + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int q = half * 256 + threadIdx.x, d = q & 63, c = (q >> 6) * 8;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = tile[c + i][d];
        if (at0 + d < length)
            storeOperand(chunkOf(turned, turned_ld, at0 + d, line0 + c, a.split), v, a.split);
    }
}

// ---- the product -------------------------------------------------------------------------------

enum { kToOperand = 0, kToTensor = 1, kToParam = 2, kToFloat = 3 };

struct Product {             // one matrix's operands, as byte offsets into its region
    int64_t a0, b0, a1, b1;  // rows of A and of B: sum over both pairs of A B^T
    int64_t e;               // the third matrix (same shape as the result), or -1
    int64_t d, dt;           // the result and its transpose, or -1
    int lda, ldb;            // bytes of a row, the same for both pairs
    int lde, ldd, lddt;
    int steps0, steps1;      // pieces of 128 bytes along each pair's rows
    int rows, cols;
};

struct GemmArgs {
    char *ws, *kept;
    const MatRec *recs;
    const Factor *factors;
    int stages, stage, symmetric, mode, split_out;
    Shapes sh;
    Product p[kMaxGroups];
};
static_assert(sizeof(GemmArgs) <= 4096, "a launch's arguments");

__device__ inline f32x16 mfma(half8 a, half8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Matrix instructions stand in groups between these two.  Without them the compiler mixes ordinary
// instructions in that write a register which the matrix instruction just before them reads.  Two earlier
// kernels were wrong exactly where the very next instruction wrote a right operand's second register, and
// right with the groups; the cause beyond that is not shown.
__device__ inline void beforeMatrix() { __builtin_amdgcn_sched_barrier(0); }
__device__ inline void afterMatrix() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 3");
    __builtin_amdgcn_sched_barrier(0);
}

// Row and column of tile number t, of all or of the lower triangle of a symmetric result: by bands
// of four rows, down the columns of each.  So a run of tiles is as square as can be, and an XCD reads
// few rows of both operands.
__device__ inline void tileOf(int t, int down, int across, bool symmetric, int &ti, int &tj) {
    constexpr int kBand = 4;
    int band;
    if (symmetric) {  // band b has kBand^2 b tiles left of its triangle, and begins at 8 b^2 + 2 b
        band = (int)((__builtin_sqrtf(8.f * (float)t + 1.f) - 1.f) * (1.f / 8.f));
        while (8 * band * band + 2 * band > t) --band;
        while (8 * (band + 1) * (band + 1) + 2 * (band + 1) <= t) ++band;
        t -= 8 * band * band + 2 * band;
        across = kBand * band;
    } else {
        band = t / (kBand * across);
        t -= band * kBand * across;
    }
    const int rows = down - kBand * band < kBand ? down - kBand * band : kBand;
    tj = t / rows;
    ti = t - tj * rows;
    if (symmetric && tj >= across) {
        t -= rows * across;
        for (tj = 0; t >= rows - tj; ++tj) t -= rows - tj;
        ti = tj + t;
        tj += across;
    }
    ti += kBand * band;
}

// The group, matrix and tile of a workgroup of the product.  Workgroups are dealt to the eight XCDs in
// turn; each of them gets an eighth of every group, in one run, so that the tiles of a matrix share
// an L2 and no XCD gets more of the long tiles than the others.
__device__ inline int findTile(const Shapes &sh, int &tile, int &mat) {
    int k = 0;
    while (k + 1 < sh.n && tile >= sh.g[k + 1].tile0) ++k;
    tile -= sh.g[k].tile0;
    const int total = sh.g[k].all, xcd = tile & 7, q = total >> 3, r = total & 7;
    tile = xcd * q + (xcd < r ? xcd : r) + (tile >> 3);
    mat = tile / sh.g[k].tiles;
    tile -= mat * sh.g[k].tiles;
    return k;
}

// 16 bytes for each lane from global memory straight into LDS: the wave's 1 KiB from `lds` on.
__device__ inline void loadToLds(const char *src, char *lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                     (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

// All but the wave's newest N loads have arrived, and so have everybody else's.
template <int N> __device__ inline void arrive() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Tile BM x BN by WM x WN waves.  A stage of LDS holds one piece of every row of both operands; STAGES
// of them are in flight, filled by loads that bypass the registers.  In LDS an operand lies as in
// memory, so a wave's read of two chunks is 1 KiB in a row.  On a full chip a 256 x 256 tile of 22-bit
// operands takes 2.5 us a piece (1.3 PFLOP/s of half products, bound by the matrix cores at the clock
// they then hold; a large half-precision matrix product of the vendor's library reaches 1.2), 4 to 5
// until the first piece is there and 9 to 12 for the stores: of the 97 us of a sum over 1024, 81 are
// products.  (A round of such tiles takes 108, with the change of workgroups.)
//
// KS > 1 (one wave to a tile) splits the sum instead: each of KS waves takes every KS-th piece and the
// partial sums are added through LDS, always in the same order.  No wave shares what it reads with
// another, so nothing goes through LDS: the pieces go from memory to the registers that the
// instructions read, kAhead of them in flight, in half the registers so that two workgroups share a
// compute unit and one's start and stores hide behind the other's sum.  P X of one 1024^2 matrix, 256
// tiles: 13 us, of which 1 is the arguments, 7 the 512 KB of every tile (it takes 3.4 at a unit's 64
// bytes a clock), 2 the partial sums and the stores; with the pieces through LDS, one workgroup to a
// unit, 15.5 (and eight matrices: 69 against 90).
template <typename T, int BM, int BN, int WM, int WN, int KS, int STAGES, bool SPLIT>
__global__ __launch_bounds__(WM *WN *KS * 64, KS > 1 ? 2 : 1) void gemm_kernel(GemmArgs a) {
    constexpr int NW = WM * WN;                          // waves that share a stage
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32;  // 32 x 32 results per wave
    constexpr int kStage = (BM + BN) * kPiece;
    constexpr int kScratch = 32 * 36 * 4;                // per wave, for the stores
    constexpr int kMain = KS > 1 ? KS * KS * 4096 : STAGES * kStage;
    constexpr int kLds = kMain > NW * KS * kScratch ? kMain : NW * KS * kScratch;
    static_assert(KS == 1 || (NW == 1 && TM * TN == KS), "one block of the sum for each wave");
    __shared__ __attribute__((aligned(16))) char lds[kLds];

    int t = blockIdx.x, mat;
    const int gi = findTile(a.sh, t, mat);
    Product p = a.p[gi];
    // (read now, all at once: what only the stores need would be waited for there, one by one)
    asm volatile("" : "+s"(p.d), "+s"(p.dt), "+s"(p.e), "+s"(p.ldd), "+s"(p.lddt), "+s"(p.rows), "+s"(p.cols));
    const Region region(a.ws, a.kept, a.sh.g[gi], mat);
    mat += a.sh.g[gi].mat0;
    int ti, tj;
    tileOf(t, (p.rows + BM - 1) / BM, (p.cols + BN - 1) / BN, a.symmetric, ti, tj);
    const int i0 = ti * BM, j0 = tj * BN;
    const int lane = threadIdx.x & 63;
    const int whole = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = KS > 1 ? 0 : whole, part = KS > 1 ? whole : 0;
    const int wi = wave / WN * (BM / WM), wj = wave % WN * (BN / WN);
    const Factor f = a.factors[(int64_t)mat * a.stages + a.stage];

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;

    // Blocks of rows beyond the matrix repeat its last one; what comes of them is not stored.
    const int last_a = (p.rows - 1) / kRows - i0 / kRows, last_b = (p.cols - 1) / kRows - j0 / kRows;
    const char *const a0 = (region + p.a0) + (int64_t)i0 * p.lda;
    const char *const b0 = (region + p.b0) + (int64_t)j0 * p.ldb;
    const char *const a1 = (region + p.a1) + (int64_t)i0 * p.lda;
    const char *const b1 = (region + p.b1) + (int64_t)j0 * p.ldb;
    // piece number k of this wave is number part + KS k of the tile
    const int steps0 = p.steps0, all = p.steps0 + p.steps1;
    const int steps = (all - part + KS - 1) / KS;
    const char *A, *B;  // the piece that is being loaded
    auto from_piece = [&](int k) {
        k = part + KS * k;
        const bool second = k >= steps0;
        const int64_t at = (int64_t)(second ? k - steps0 : k) * (kRows * kPiece);
        A = (second ? a1 : a0) + at;
        B = (second ? b1 : b0) + at;
    };
    // before the second pair's first product
    bool turned_sum = all == steps0;
    auto turn = [&] {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] *= f.turn;
        turned_sum = true;
    };

    if constexpr (KS > 1) {
        constexpr int kAhead = STAGES;
        unsigned from_a[TM], from_b[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
            from_a[i] = (unsigned)(i < last_a ? i : last_a) * (unsigned)(kRows * p.lda) + lane * 16;
#pragma unroll
        for (int j = 0; j < TN; ++j)
            from_b[j] = (unsigned)(j < last_b ? j : last_b) * (unsigned)(kRows * p.ldb) + lane * 16;
        half8 xa[kAhead][TM][4], xb[kAhead][TN][4];  // chunks 0 2 4 6 of a piece
        auto fetch = [&](int k, int to) {
            from_piece(k);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
#pragma unroll
                for (int i = 0; i < TM; ++i) xa[to][i][q] = *global<half8>(A + from_a[i] + q * 1024);
#pragma unroll
                for (int j = 0; j < TN; ++j) xb[to][j][q] = *global<half8>(B + from_b[j] + q * 1024);
            }
        };
        auto multiply = [&](int k, int from) {
            if (!turned_sum && part + KS * k >= steps0) turn();
            auto each = [&](int q, int r) {
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        acc[i][j] = mfma(xa[from][i][q], xb[from][j][r], acc[i][j]);
            };
            beforeMatrix();
            each(0, 0);
            each(1, 1);
            if (SPLIT) {
                each(2, 0);
                each(3, 1);
                each(0, 2);
                each(1, 3);
            } else {
                each(2, 2);
                each(3, 3);
            }
            afterMatrix();
        };
        // (whole rounds have no condition inside and are reached by one way only, so that the waits
        // are for the oldest loads alone)
        if (steps >= kAhead) {
#pragma unroll
            for (int d = 0; d < kAhead; ++d) fetch(d, d);
            int k = 0;
            for (; k + 2 * kAhead <= steps; k += kAhead) {
#pragma unroll
                for (int d = 0; d < kAhead; ++d) {
                    multiply(k + d, d);
                    fetch(k + d + kAhead, d);
                }
            }
#pragma unroll
            for (int d = 0; d < 2 * kAhead - 1; ++d) {
                if (d >= kAhead && k + d >= steps) break;
                multiply(k + d, d % kAhead);
                if (d < kAhead - 1 && k + d + kAhead < steps) fetch(k + d + kAhead, d);
            }
        } else {
#pragma unroll
            for (int d = 0; d < kAhead - 1; ++d)
                if (d < steps) fetch(d, d);
#pragma unroll
            for (int d = 0; d < kAhead - 1; ++d)
                if (d < steps) multiply(d, d);
        }
    } else {
        constexpr int LA = BM / 8 / NW, LB = BN / 8 / NW;  // loads of 1 KiB, per wave and stage
        unsigned from_a[LA], from_b[LB];
#pragma unroll
        for (int q = 0; q < LA; ++q) {
            const int n = q * NW + wave, block = n / 4;
            from_a[q] = (unsigned)(block < last_a ? block : last_a) * (unsigned)(kRows * p.lda) +
                        n % 4 * 1024 + lane * 16;
        }
#pragma unroll
        for (int q = 0; q < LB; ++q) {
            const int n = q * NW + wave, block = n / 4;
            from_b[q] = (unsigned)(block < last_b ? block : last_b) * (unsigned)(kRows * p.ldb) +
                        n % 4 * 1024 + lane * 16;
        }
        auto load = [&](int q, int stage) {
            char *to = lds + stage * kStage;
            if (q < LA)
                loadToLds(A + from_a[q < LA ? q : 0], to + (q * NW + wave) * 1024);
            else
                loadToLds(B + from_b[q < LA ? 0 : q - LA],
                          to + BM * kPiece + ((q - LA) * NW + wave) * 1024);
        };
        // Phases of TM * TN matrix instructions.  The registers of a phase are read from LDS during
        // the one before.  Before a step's last phase everybody has read the stage and the next one
        // is waited for; the last phase's instructions cover the first reads from that one, and the
        // loads that refill the stage go out in the last phase and the kShares - 1 that follow it.
        constexpr int kShares = SPLIT ? 3 : 2, L = LA + LB, kFirst = (L + kShares - 1) / kShares;
        half8 ah[2][TM], bh[2][TN], al[SPLIT ? TM : 1], bl[SPLIT ? TN : 1];
        auto read_a = [&](const char *from, half8 *to, int c) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
                to[i] = *(const half8 *)(from + (wi + 32 * i) * kPiece + c * 512 + lane * 16);
        };
        auto read_b = [&](const char *from, half8 *to, int c) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
                to[j] = *(const half8 *)(from + (BM + wj + 32 * j) * kPiece + c * 512 + lane * 16);
        };
        auto multiply = [&](const half8 *x, const half8 *y) {
            beforeMatrix();
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = mfma(x[i], y[j], acc[i][j]);
            afterMatrix();
        };
        // share number `share` of the loads of the piece that `from_piece` chose
        auto refill = [&](int share, int stage) {
#pragma unroll
            for (int q = 0; q < L; ++q)
                if (q / kFirst == share) load(q, stage);
        };
#pragma unroll
        for (int k = 0; k < STAGES; ++k) {
            if (k >= steps) break;
            from_piece(k);
#pragma unroll
            for (int share = 0; share < (k == STAGES - 1 ? 1 : kShares); ++share) refill(share, k);
        }
        if (steps >= STAGES)
            arrive<(STAGES - 2) * L + kFirst>();
        else
            arrive<0>();
        read_a(lds, ah[0], 0);
        read_b(lds, bh[0], 0);
        int stage = 0;
        for (int k = 0; k < steps; ++k) {
            const char *const here = lds + stage * kStage;
            const int next = stage == STAGES - 1 ? 0 : stage + 1;
            const int before = stage == 0 ? STAGES - 1 : stage - 1;  // being refilled
            const bool filling = k + STAGES - 1 < steps;
            if (!turned_sum && k >= steps0) turn();
            __builtin_amdgcn_sched_barrier(0);
            if (SPLIT) {
                read_a(here, al, 4);
                if (filling) refill(1, before);
                multiply(ah[0], bh[0]);
                read_b(here, bl, 4);
                if (filling) refill(2, before);
                multiply(al, bh[0]);
                read_a(here, ah[1], 2);
                read_b(here, bh[1], 2);
                multiply(ah[0], bl);
                read_a(here, al, 6);
                multiply(ah[1], bh[1]);
                read_b(here, bl, 6);
                multiply(al, bh[1]);
            } else {
                read_a(here, ah[1], 2);
                read_b(here, bh[1], 2);
                if (filling) refill(1, before);
                multiply(ah[0], bh[0]);
                read_a(here, ah[0], 4);
                read_b(here, bh[0], 4);
                multiply(ah[1], bh[1]);
                read_a(here, ah[1], 6);
                read_b(here, bh[1], 6);
                multiply(ah[0], bh[0]);
            }
            // (towards the end fewer pieces are in flight: everything is waited for)
            if (filling)
                arrive<(STAGES - 2) * L>();
            else
                arrive<0>();
            read_a(lds + next * kStage, ah[0], 0);
            read_b(lds + next * kStage, bh[0], 0);
            if (k + STAGES < steps) {
                from_piece(k + STAGES);
                refill(0, stage);
            }
            if (SPLIT)
                multiply(ah[1], bl);
            else
                multiply(ah[1], bh[1]);
            stage = next;
        }
        arrive<0>();
    }
    if (!turned_sum) turn();  // (a wave that had no piece of the second pair)
    if constexpr (KS > 1) {
        // each wave adds up one block
        f32x4 *const sums = (f32x4 *)lds;
        auto at = [&](int block, int from, int q) { return ((block * KS + from) * 4 + q) * 64 + lane; };
#pragma unroll
        for (int b = 0; b < KS; ++b) {
            if (b == whole) continue;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x16 &s = acc[b / TN][b % TN];
                sums[at(b, whole, q)] = f32x4{s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
            }
        }
        __syncthreads();
        f32x16 sum, own;
#pragma unroll
        for (int b = 0; b < KS; ++b)
            if (b == whole) own = acc[b / TN][b % TN];
#pragma unroll
        for (int w = 0; w < KS; ++w) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 s = sums[at(whole, w == whole ? 0 : w, q)];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = w == whole ? own[4 * q + i] : s[i];
                    sum[4 * q + i] = w ? sum[4 * q + i] + v : v;
                }
            }
        }
#pragma unroll
        for (int b = 0; b < KS; ++b)
            if (b == whole) acc[b / TN][b % TN] = sum;
        __syncthreads();
    }

    // Results leave by 32 x 32 blocks.  A lane has four times four neighbours of one column: halves of
    // chunks of the transpose, which is stored as it is; by rows they go through LDS, as the two halves
    // they end as.  (Instructions count here, up to eight blocks to a wave: what only some blocks need
    // stands behind a branch.)
    float *box = (float *)(lds + whole * kScratch);
    const MatRec &r = a.recs[mat];
    const bool tensor = a.mode == kToTensor || a.mode == kToParam;
    const bool turned = tensor && r.out_rs < r.out_cs;
    const bool mirror = p.dt >= 0 && !(a.symmetric && ti == tj);
    for (int block = KS > 1 ? whole : 0; block < (KS > 1 ? whole + 1 : TM * TN); ++block) {
        const int bi = i0 + wi + block / TN * 32, bj = j0 + wj + block % TN * 32;
        if (bi >= p.rows && !(p.dt >= 0 && bi < padded(p.rows))) continue;
        if (bj >= p.cols && !(p.d >= 0 && bj < padded(p.cols))) continue;
        const int col = bj + (lane & 31), row0 = bi + (lane >> 5) * 4;  // and rows (q / 4) * 8 + q % 4 on
        // (registers are picked by number: every block has its own, the rest is shared code)
        float v[16];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                if (block == i * TN + j)
#pragma unroll
                    for (int q = 0; q < 16; ++q) v[q] = acc[i][j][q] * f.acc;
        // (the third matrix is symmetric, so it can be read as the transpose is stored)
        if (p.e >= 0 && col < p.cols) {
            const char *from = chunkOf(region + p.e, p.lde, col, bi, SPLIT) + (lane >> 5) * 8;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const half4 hi = *global<half4>(from + q * 512);
                half4 lo = {};
                if (SPLIT) lo = *global<half4>(from + q * 512 + 2048);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * q + i] += f.add * ((float)hi[i] + (float)lo[i]);
            }
        }
        if (bi == bj && f.diag != 0.f) {
#pragma unroll
            for (int q = 0; q < 16; ++q)
                if (row0 + (q >> 2) * 8 + (q & 3) == col) v[q] += f.diag;
        }
        if (bi + 32 > p.rows || bj + 32 > p.cols) {
#pragma unroll
            for (int q = 0; q < 16; ++q)
                if (row0 + (q >> 2) * 8 + (q & 3) >= p.rows || col >= p.cols) v[q] = 0.f;
        }
        const int box_at = (lane >> 5) * 4 * 36 + (lane & 31);
        if (a.mode == kToOperand) {
            unsigned u[16];  // low 16 bits: hi; high 16 bits: lo
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const _Float16 hi = (_Float16)v[q];
                const _Float16 lo = (_Float16)__builtin_fmaf((float)hi, -1.f, v[q]);
                u[q] = __builtin_bit_cast(unsigned short, hi) |
                       (unsigned)__builtin_bit_cast(unsigned short, lo) << 16;
            }
            auto his = [](unsigned x, unsigned y) { return __builtin_amdgcn_perm(y, x, 0x05040100); };
            auto los = [](unsigned x, unsigned y) { return __builtin_amdgcn_perm(y, x, 0x07060302); };
            if (mirror && col < p.cols) {
                char *to = chunkOf(region + p.dt, p.lddt, col, bi, a.split_out) + (lane >> 5) * 8;
#pragma unroll
                for (int q = 0; q < 16; q += 4)
                    *global<u32x2>(to + q * 128) = u32x2{his(u[q], u[q + 1]), his(u[q + 2], u[q + 3])};
                if (a.split_out)
#pragma unroll
                    for (int q = 0; q < 16; q += 4)
                        *global<u32x2>(to + q * 128 + 2048) =
                            u32x2{los(u[q], u[q + 1]), los(u[q + 2], u[q + 3])};
            }
            if (p.d < 0) continue;
            unsigned *const ubox = (unsigned *)box;
#pragma unroll
            for (int q = 0; q < 16; ++q) ubox[box_at + ((q >> 2) * 8 + (q & 3)) * 36] = u[q];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int row = lane & 31, c = (lane >> 5) * 8;
            char *to = chunkOf(region + p.d, p.ldd, bi + row, bj, a.split_out) + c * 64;
            unsigned x[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) x[q] = ubox[row * 36 + c + (q >> 3) * 16 + (q & 7)];
            if (bi + row < p.rows) {
#pragma unroll
                for (int q = 0; q < 16; q += 8) {
                    const unsigned *y = x + q;
                    *global<u32x4>(to + q * 128) = u32x4{his(y[0], y[1]), his(y[2], y[3]),
                                                         his(y[4], y[5]), his(y[6], y[7])};
                    if (a.split_out)
                        *global<u32x4>(to + q * 128 + 2048) = u32x4{los(y[0], y[1]), los(y[2], y[3]),
                                                                    los(y[4], y[5]), los(y[6], y[7])};
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            continue;
        }
#pragma unroll
        for (int q = 0; q < 16; ++q) box[box_at + ((q >> 2) * 8 + (q & 3)) * 36] = v[q];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float x[8], e[8];
            // eight neighbours of the caller's tensor, along the way it lies
            const int line = half * 16 + (lane >> 2), c = (lane & 3) * 8;
            const int row = bi + (turned ? c : line), column = bj + (turned ? line : c);
            if (row >= p.rows || column >= p.cols) continue;
#pragma unroll
            for (int q = 0; q < 8; ++q) x[q] = turned ? box[(c + q) * 36 + line] : box[line * 36 + c + q];
            const int valid = turned ? p.rows - row : p.cols - column;
            if (a.mode == kToFloat) {
                store8((float *)((region + p.d) + (int64_t)row * p.ldd) + column, valid, x);
                continue;
            }
            T *o = (T *)r.out + row * r.out_rs + column * r.out_cs;
            const int64_t by = turned ? r.out_rs : r.out_cs;
            if (by == 1) {
                if (a.mode == kToParam) {
                    load8(o, valid, e);
#pragma unroll
                    for (int q = 0; q < 8; ++q) x[q] = r.keep * e[q] - r.rate * x[q];
                } else {
#pragma unroll
                    for (int q = 0; q < 8; ++q) x[q] *= r.rate;
                }
                store8(o, valid, x);
            } else {
                for (int q = 0; q < 8 && q < valid; ++q) {
                    TOA_GLOBAL T *y = global<T>((void *)(o + q * by));
                    *y = fromFloat<T>(a.mode == kToParam ? r.keep * toFloat(*y) - r.rate * x[q]
                                                         : r.rate * x[q]);
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- thin matrices -----------------------------------------------------------------------------
//
// Two steps at once are five products of s x s matrices between one of X with itself and one with X.
// With up to 64 rows each of the five is a single tile, so one workgroup makes all of them for a
// matrix, from S to Q, in LDS: four waves, a 32 x 32 block each.  Bound by the way through five
// products in a row: 14 us where five launches take 29 (one 32 x 2048 float32 matrix: 114 -> 83 us, 24
// of 60 x 1500: 140 -> 107).

constexpr int kThin = 64;

struct SquareArgs {
    char *ws;
    const Factor *factors;
    int stages, stage;
    Shapes sh;
    int64_t off[kMaxGroups];  // of S, and then of Q
};

__global__ __launch_bounds__(256) void square_kernel(SquareArgs a) {
    constexpr int kBlock32 = kRows * kThin * 4;  // bytes of 32 rows: two pieces
    __shared__ __attribute__((aligned(16))) char lds[3][2 * kBlock32];
    int part = blockIdx.x, mat;
    const int gi = findGroup(a.sh, part, mat);
    const Group &g = a.sh.g[gi];
    char *const global_s = Region(a.ws, a.ws, g, mat) + a.off[gi];
    mat += g.mat0;
    const int s = g.s;
    const Factor *const f = a.factors + (int64_t)mat * a.stages + a.stage;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int p = wave >> 1, q = wave & 1;
    // (16 bytes are a chunk of one row; rows beyond the matrix hold anything)
    for (int i = threadIdx.x; i < 2 * kBlock32 / 16; i += 256) {
        const int row = i / (kBlock32 / 16) * kRows + i % kRows;
        half8 v = {};
        if (row < s) v = *global<half8>(global_s + i * 16);
        *(half8 *)(lds[0] + i * 16) = v;
    }
    __syncthreads();
    // D = f.acc A B^T + f.add E + f.diag I, all of them symmetric: the result is written as its transpose
    const int mine = q * kBlock32 + p * (kRows * kPiece) + (lane & 31) * 16 + (lane >> 5) * 8;
    auto product = [&](const char *A, const char *B, const char *E, char *D, const Factor f) {
        f32x16 sum;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[i] = 0.f;
#pragma unroll
        for (int piece = 0; piece < 2; ++piece) {
            half8 x[4], y[4];  // two of hi, two of lo
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int at = piece * kRows * kPiece + c * 1024 + lane * 16;
                x[c] = *(const half8 *)(A + p * kBlock32 + at);
                y[c] = *(const half8 *)(B + q * kBlock32 + at);
            }
            beforeMatrix();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                sum = mfma(x[2 + c], y[c], sum);
                sum = mfma(x[c], y[2 + c], sum);
                sum = mfma(x[c], y[c], sum);
            }
            afterMatrix();
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            half4 hi, lo, eh = {}, el = {};
            if (f.add != 0.f) {
                eh = *(const half4 *)(E + mine + u * 512);
                el = *(const half4 *)(E + mine + u * 512 + 2048);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = p * 32 + u * 8 + (lane >> 5) * 4 + i, col = q * 32 + (lane & 31);
                float v = sum[4 * u + i] * f.acc;
                if (f.add != 0.f) v += f.add * ((float)eh[i] + (float)el[i]);
                if (row == col) v += f.diag;
                if (row >= s || col >= s) v = 0.f;
                hi[i] = (_Float16)v;
                lo[i] = (_Float16)(v - (float)hi[i]);
            }
            *(half4 *)(D + mine + u * 512) = hi;
            *(half4 *)(D + mine + u * 512 + 2048) = lo;
        }
        __syncthreads();
    };
    char *const S = lds[0], *const P = lds[1], *const T = lds[2];
    product(S, S, S, P, f[1]);
    product(P, S, S, T, f[2]);
    product(T, P, S, S, f[3]);
    product(S, S, S, T, f[4]);
    product(T, P, S, S, f[5]);
    for (int i = threadIdx.x; i < (s + kRows - 1) / kRows * (kBlock32 / 16); i += 256)
        *global<half8>(global_s + i * 16) = *(const half8 *)(S + i * 16);
}

// ---- small matrices ----------------------------------------------------------------------------
//
// Up to 32 rows and 864 columns, or 64 and 224: one workgroup takes a matrix through everything, and
// the iterates never leave its LDS.  What a small matrix costs is not arithmetic but the way through
// nineteen launches: three float32 ones of 32 x 288 take 24 us here and 125 through the tiles, with their
// gradient 85 and 389.  Of the 24, 5 are the norm and the factors, 6 the way into LDS, 2.4 each step, of
// which the sums over the waves take most.
//
// Eight waves share the columns by blocks of 32.  A block's result of a matrix instruction has a
// column in each lane and rows in its registers (layout C); that is just the layout of the right
// operand of P X -- the order of the rows within the sum is another one, but P can be read in the
// same order.  The other way round, X^T P gives rows in the lanes and columns in the registers
// (layout R), which is what X X^T wants of both its operands.  So each product is made twice, once
// in each layout, and nothing is ever transposed.

constexpr int kSmallWaves = 8;
constexpr int kSmallInline = 24;  // records that fit in a launch's arguments

struct SmallArgs {
    Series q;
    StepArgs step;
    const MatRec *recs;  // or null: the records below
    char *ws;            // gradient: the iterates, `stride` bytes for each matrix
    int64_t stride;
    int apply;
    MatRec r[kSmallInline];
};

__host__ __device__ constexpr int smallRow(int rb) { return rb * 128 + 8; }  // (8: rows 32 lanes apart hit other banks)

// Bytes the gradient keeps of one step: both layouts of every block of 32 columns, and S.
__host__ __device__ constexpr int64_t smallKept(int rb, int w) {
    return (int64_t)((w + 31) / 32) * rb * 2 * 4096 + (int64_t)rb * 32 * smallRow(rb);
}

// 16 values of a layout as operand registers: hi and lo for each half of the sum.
struct Pair {
    half8 hi[2], lo[2];
    __device__ void set(const f32x16 &v) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            hi[i >> 3][i & 7] = (_Float16)v[i];
            // (v - hi, which is exact, as the one instruction that reads a half in place)
            lo[i >> 3][i & 7] = (_Float16)__builtin_fmaf((float)hi[i >> 3][i & 7], -1.f, v[i]);
        }
    }
    __device__ float value(int i) const { return (float)hi[i >> 3][i & 7] + (float)lo[i >> 3][i & 7]; }
};

// ALL: with lo lo, for float32 (see the top).
template <bool ALL> __device__ inline f32x16 product(const Pair &a, const Pair &b, f32x16 sum) {
    beforeMatrix();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        if (ALL) sum = mfma(a.lo[t], b.lo[t], sum);
        sum = mfma(a.lo[t], b.hi[t], sum);
        sum = mfma(a.hi[t], b.lo[t], sum);
        sum = mfma(a.hi[t], b.hi[t], sum);
    }
    afterMatrix();
    return sum;
}

// p x into one sum and x p into another, by turns: neither waits for its own last result.
template <bool ALL>
__device__ inline void productBoth(const Pair &p, const Pair &x, f32x16 &px, f32x16 &xp) {
    beforeMatrix();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        if (ALL) {
            px = mfma(p.lo[t], x.lo[t], px);
            xp = mfma(x.lo[t], p.lo[t], xp);
        }
        px = mfma(p.lo[t], x.hi[t], px);
        xp = mfma(x.hi[t], p.lo[t], xp);
        px = mfma(p.hi[t], x.lo[t], px);
        xp = mfma(x.lo[t], p.hi[t], xp);
        px = mfma(p.hi[t], x.hi[t], px);
        xp = mfma(x.hi[t], p.hi[t], xp);
    }
    afterMatrix();
}

__device__ inline f32x16 zero16() {
    f32x16 v;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.f;
    return v;
}

// Row (layout C) or column (layout R) within a block of register i.
__device__ inline int laneRow(int i, int lane) { return (i >> 2) * 8 + (lane >> 5) * 4 + (i & 3); }

// Block (r, k) of a symmetric matrix in LDS as an operand, its sum in the order of laneRow.
template <int RB> __device__ inline Pair readSymmetric(const char *m, int r, int k, int lane) {
    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
    const char *row = m + (r * 32 + (lane & 31)) * smallRow(RB) + k * 128 + (lane >> 5) * 8;
    Pair p;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const half4 hi = *(const half4 *)(row + (2 * t + u) * 16);
            const half4 lo = *(const half4 *)(row + 64 + (2 * t + u) * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p.hi[t][4 * u + i] = hi[i];
                p.lo[t][4 * u + i] = lo[i];
            }
        }
    return p;
}

template <int RB> __device__ inline void writeElement(char *m, int row, int col, float v) {
    _Float16 *p = (_Float16 *)(m + row * smallRow(RB) + (col >> 5) * 128) + (col & 31);
    const _Float16 hi = (_Float16)v;
    p[0] = hi;
    p[32] = (_Float16)(v - (float)hi);
}

// A result block of a symmetric matrix (layout C) into LDS, with its mirror image.
template <int RB>
__device__ inline void writeSymmetric(char *m, int r, int k, int lane, const f32x16 &v, const Factor &f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int row = r * 32 + laneRow(i, lane), col = k * 32 + (lane & 31);
        const float x = v[i] * f.acc + (row == col ? f.diag : 0.f);
        writeElement<RB>(m, row, col, x);
        if (r != k) writeElement<RB>(m, col, row, x);
    }
}

// Adds up the waves' shares of a symmetric matrix (lower blocks, always in the same order) into LDS.
// With 64 rows there is LDS for the shares of four waves: the others' are added to theirs first.
constexpr int smallSlots(int rb) { return rb == 1 ? kSmallWaves : kSmallWaves / 2; }

template <int RB>
__device__ inline void gather(f32x16 (&share)[RB * (RB + 1) / 2], float *shares, char *m,
                              const Factor &f) {
    constexpr int kBlocks = RB * (RB + 1) / 2, kSlots = smallSlots(RB);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto put = [&](int slot) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) shares[((b * kSlots + slot) * 16 + i) * 64 + lane] = share[b][i];
    };
    if (kSlots < kSmallWaves) {
        if (wave >= kSlots) put(wave - kSlots);
        __syncthreads();
        if (wave < kSlots) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    share[b][i] += shares[((b * kSlots + wave) * 16 + i) * 64 + lane];
        }
    }
    if (wave < kSlots) put(wave);
    __syncthreads();
    for (int e = threadIdx.x; e < kBlocks * 1024; e += kSmallWaves * 64) {
        const int b = e >> 10, x = e & 1023;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kSlots; ++w) v += shares[(b * kSlots + w) * 1024 + x];
        const int r = b ? 1 : 0, k = b == 2 ? 1 : 0;  // (0,0), (1,0), (1,1)
        const int row = r * 32 + laneRow(x >> 6, x & 63), col = k * 32 + (x & 31);
        v = v * f.acc + (row == col ? f.diag : 0.f);
        writeElement<RB>(m, row, col, v);
        if (r != k) writeElement<RB>(m, col, row, v);
    }
    __syncthreads();
}

constexpr int smallColumnBlocks(int rb) { return rb == 1 ? 27 : 7; }

template <typename T, int KIND, int RB, bool BACK>
__global__ __launch_bounds__(kSmallWaves * 64) void small_kernel(SmallArgs a) {
    using Word = half8;
    constexpr int kBlocks = RB * (RB + 1) / 2, kMatrix = RB * 32 * smallRow(RB);
    __shared__ Word X[smallColumnBlocks(RB) * RB * 256];
    __shared__ float shares[kBlocks * smallSlots(RB) * 1024];
    __shared__ __attribute__((aligned(16))) char S[kMatrix], P[kMatrix], M[BACK ? kMatrix : 16];
    __shared__ Factor factors[(BACK ? 6 : 3) * kMaxSteps];
    __shared__ double sums[kSmallWaves];
    __shared__ SeriesTable table;

    constexpr bool kAll = std::is_same<T, float>::value;
    auto multiply = [](const Pair &x, const Pair &y, const f32x16 &sum) { return product<kAll>(x, y, sum); };
    auto multiplyBoth = [](const Pair &p, const Pair &x, f32x16 &px, f32x16 &xp) {
        productBoth<kAll>(p, x, px, xp);
    };
    const MatRec r = uniform(a.recs ? a.recs + blockIdx.x : a.r + blockIdx.x);
    const int s = r.s, w = r.w, steps = a.q.steps;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n = (int64_t)s * w;
    char *kept = BACK ? a.ws + blockIdx.x * a.stride : nullptr;
    table.load(a.q);

    constexpr int kSum = KIND == kPackG ? kSumG : KIND == kPackM ? kMomentum
                         : KIND == kPackMF32 ? kMomentumF32 : kMomentumI8;
    const double size = sqrt(blockSum(sumPass<T, kSum>(r, a.step, 0, n), sums));
    const double ysize = BACK ? sqrt(blockSum(sumPass<T, kSumAux>(r, a.step, 0, n), sums)) : 0.0;
    const Bounds bounds(a.q, table, size, ysize);
    const MatNorm norm = normOf(bounds, size);
    if ((int)threadIdx.x < steps)
        stepFactors(bounds, threadIdx.x, factors + 3 * threadIdx.x,
                    BACK ? factors + 3 * (steps + threadIdx.x) : nullptr);
    __syncthreads();

    const int blocks = (w + 31) / 32;  // this wave's are number `wave`, wave + 8, ...
    auto load = [&](auto kind, double scale, int b, int rb, bool by_rows) {
        constexpr int kKind = decltype(kind)::value;
        // a lane's first element, and the way to the others, which is the same for all lanes
        const int row0 = rb * 32 + (by_rows ? lane & 31 : (lane >> 5) * 4);
        const int j0 = b * 32 + (by_rows ? (lane >> 5) * 4 : lane & 31);
        const int64_t rs = kKind == kPackAux ? r.aux_rs : r.g_rs, cs = kKind == kPackAux ? r.aux_cs : r.g_cs;
        const int64_t at0 = row0 * rs + j0 * cs, by = by_rows ? cs : rs;
        const int left = by_rows ? w - j0 : s - row0;  // elements along the registers
        const bool inside = by_rows ? row0 < s : j0 < w;
        f32x16 v;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int along = (i >> 2) * 8 + (i & 3);
            const bool valid = inside && along < left;
            // (read in any case, element 0 if need be: a branch would wait for every one in turn)
            const float e = element<T, kKind>(r, a.step, valid ? at0 + along * by : 0);
            v[i] = valid ? (float)((double)e * scale) : 0.f;
        }
        return v;
    };
    // registers in LDS, and (the gradient's iterates) in the workspace: 16 bytes of each lane in turn
    auto putPair = [&](auto *to, const Pair &p) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            to[t * 64 + lane] = p.hi[t];
            to[(2 + t) * 64 + lane] = p.lo[t];
        }
    };
    auto getPair = [&](const auto *from) {
        Pair p;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            p.hi[t] = from[t * 64 + lane];
            p.lo[t] = from[(2 + t) * 64 + lane];
        }
        return p;
    };
    auto inLds = [&](int b, int rb) { return X + (b * RB + rb) * 256; };
    auto inKept = [&](int k, int b, int rb, int layout) {
        return global<Word>((void *)(kept + k * smallKept(RB, w) +
                                     (((int64_t)b * RB + rb) * 2 + layout) * 4096));
    };
    auto inKeptS = [&](int k) {
        return global<int64_t>((void *)(kept + (k + 1) * smallKept(RB, w) - kMatrix));
    };
    auto copyMatrix = [&](auto *to, const auto *from) {
        for (int i = threadIdx.x; i < kMatrix / 8; i += kSmallWaves * 64) to[i] = from[i];
    };

    using Main = std::integral_constant<int, KIND>;
    f32x16 share[kBlocks];
    auto clear = [&] {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) share[b] = zero16();
    };
    // adds a block's part of X X^T
    auto addGram = [&](const Pair (&l)[RB]) {
#pragma unroll
        for (int p = 0; p < RB; ++p)
#pragma unroll
            for (int q = 0; q <= p; ++q)
                share[p * (p + 1) / 2 + q] = multiply(l[p], l[q], share[p * (p + 1) / 2 + q]);
    };
    clear();
#pragma unroll 1
    for (int b = wave; b < blocks; b += kSmallWaves) {
        Pair l[RB];
#pragma unroll
        for (int p = 0; p < RB; ++p) {
            Pair c;
            c.set(load(Main(), norm.x_scale, b, p, false));
            l[p].set(load(Main(), norm.x_scale, b, p, true));
            putPair(inLds(b, p), c);
            if (BACK) {
                putPair(inKept(0, b, p, 0), c);
                putPair(inKept(0, b, p, 1), l[p]);
            }
        }
        addGram(l);
    }
    // the block of a symmetric result that a wave makes
    const int bp = wave ? 1 : 0, bq = wave == 2 ? 1 : 0;
    // v * f.acc + f.add * (block of m)
    auto withThird = [&](f32x16 v, const char *m, const Factor &f) {
        v *= f.acc;
        if (f.add != 0.f) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const _Float16 *e =
                    (const _Float16 *)(m + ((RB == 1 ? 0 : bp * 32) + laneRow(i, lane)) * smallRow(RB) +
                                       (RB == 1 ? 0 : bq * 128)) + (lane & 31);
                v[i] += f.add * ((float)e[0] + (float)e[32]);
            }
        }
        return v;
    };
    // P from S.  With one block every wave makes it for itself: a result of a symmetric product is
    // an operand as it stands (lanes and registers change places).  With four they share the work.
    Pair own_p, own_n;
    auto asOperand = [&](f32x16 v, float diag) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] += laneRow(i, lane) == (lane & 31) ? diag : 0.f;
        Pair p;
        p.set(v);
        return p;
    };
    auto makeP = [&](const Factor &f) {
        if (RB == 1) {
            const Pair e = readSymmetric<RB>(S, 0, 0, lane);
            own_p = asOperand(withThird(multiply(e, e, zero16()), S, f), f.diag);
        } else {
            if (wave < kBlocks) {
                f32x16 v = zero16();
#pragma unroll
                for (int e = 0; e < RB; ++e)
                    v = multiply(readSymmetric<RB>(S, bp, e, lane), readSymmetric<RB>(S, bq, e, lane), v);
                writeSymmetric<RB>(P, bp, bq, lane, withThird(v, S, f), {1.f, 0.f, 1.f, f.diag});
            }
            __syncthreads();
        }
    };
    auto operandP = [&](int p, int e) { return RB == 1 ? own_p : readSymmetric<RB>(P, p, e, lane); };
#pragma unroll 1
    for (int k = 0; k < steps; ++k) {
        const Factor f0 = factors[3 * k], f1 = factors[3 * k + 1], f2 = factors[3 * k + 2];
        const bool last = k + 1 == steps;
        gather<RB>(share, shares, S, f0);
        makeP(f1);
        if (BACK) {
            copyMatrix(inKeptS(k), (const int64_t *)S);
            if (last) break;
        }
        clear();
#pragma unroll 1
        for (int b = wave; b < blocks; b += kSmallWaves) {
            Pair x[RB], l[RB];
#pragma unroll
            for (int p = 0; p < RB; ++p) x[p] = getPair(inLds(b, p));
#pragma unroll
            for (int p = 0; p < RB; ++p) {
                f32x16 vc = zero16(), vr = zero16();
#pragma unroll
                for (int e = 0; e < RB; ++e) {
                    const Pair pe = operandP(p, e);
                    if (last)
                        vc = multiply(pe, x[e], vc);
                    else
                        multiplyBoth(pe, x[e], vc, vr);
                }
                vc *= f2.acc;
                if (last) {
                    const int j = b * 32 + (lane & 31);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int row = p * 32 + laneRow(i, lane);
                        TOA_GLOBAL T *o = global<T>(r.out) + (row < s ? row : s - 1) * r.out_rs +
                                          (j < w ? j : w - 1) * r.out_cs;
                        float v = r.rate * vc[i];
                        if (a.apply) v = r.keep * toFloat(*o) - v;
                        if (row < s && j < w) *o = fromFloat<T>(v);
                    }
                } else {
                    Pair c;
                    c.set(vc);
                    putPair(inLds(b, p), c);  // (x has been read)
                    l[p].set(vr * f2.acc);
                    if (BACK) {
                        putPair(inKept(k + 1, b, p, 0), c);
                        putPair(inKept(k + 1, b, p, 1), l[p]);
                    }
                }
            }
            if (!last) addGram(l);
        }
    }
    if (!BACK) return;

    // The way back: X holds the cotangent Y in layout C, share its part of Y X^T + X Y^T.
    using Aux = std::integral_constant<int, kPackAux>;
    auto addBoth = [&](const Pair (&y)[RB], const Pair (&l)[RB]) {
#pragma unroll
        for (int p = 0; p < RB; ++p)
#pragma unroll
            for (int q = 0; q <= p; ++q) {
                f32x16 &v = share[p * (p + 1) / 2 + q];
                v = multiply(y[p], l[q], v);
                v = multiply(l[p], y[q], v);
            }
    };
    clear();
#pragma unroll 1
    for (int b = wave; b < blocks; b += kSmallWaves) {
        Pair l[RB];
#pragma unroll
        for (int p = 0; p < RB; ++p) {
            Pair c;
            c.set(load(Aux(), norm.y_scale, b, p, false));
            l[p].set(load(Aux(), norm.y_scale, b, p, true));
            putPair(inLds(b, p), c);
        }
        Pair xr[RB];
#pragma unroll
        for (int p = 0; p < RB; ++p) xr[p] = getPair(inKept(steps - 1, b, p, 1));
        addBoth(l, xr);
    }
    // both layouts of a block of X_k and X_k-1, from the workspace: asked for well before their use
    Pair next_c[RB], next_r[RB];
    auto prefetch = [&](int k, int b) {
        if (RB > 1 || b >= blocks) return;  // (two rows of blocks leave no registers for it)
#pragma unroll
        for (int p = 0; p < RB; ++p) {
            next_c[p] = getPair(inKept(k, b, p, 0));
            if (k) next_r[p] = getPair(inKept(k - 1, b, p, 1));
        }
    };
    double dot = 0.0;
#pragma unroll 1
    for (int k = steps - 1; k >= 0; --k) {
        const Factor f0 = factors[3 * (steps + k)], f1 = factors[3 * (steps + k) + 1],
                     f2 = factors[3 * (steps + k) + 2];
        prefetch(k, wave);
        __syncthreads();  // S, P and M of the step before are no longer read
        copyMatrix((int64_t *)S, inKeptS(k));
        gather<RB>(share, shares, M, f0);
        if (k + 1 < steps) makeP(factors[3 * k + 1]);  // (the last step's is still there)
        f32x16 v = zero16();
        if (RB == 1 || wave < kBlocks) {
#pragma unroll
            for (int e = 0; e < RB; ++e) {
                const int p = RB == 1 ? 0 : bp, q = RB == 1 ? 0 : bq;
                v = multiply(readSymmetric<RB>(M, p, e, lane), readSymmetric<RB>(S, q, e, lane), v);
                v = multiply(readSymmetric<RB>(S, p, e, lane), readSymmetric<RB>(M, q, e, lane), v);
            }
            v = withThird(v, M, f1);
        }
        if (RB == 1) {
            own_n.set(v);
        } else {
            __syncthreads();
            if (wave < kBlocks) writeSymmetric<RB>(M, bp, bq, lane, v, {1.f, 0.f, 1.f, 0.f});  // N
            __syncthreads();
        }
        clear();
#pragma unroll 1
        for (int b = wave; b < blocks; b += kSmallWaves) {
            Pair y[RB], x[RB], xr[RB], l[RB];
#pragma unroll
            for (int e = 0; e < RB; ++e) {
                y[e] = getPair(inLds(b, e));
                x[e] = RB > 1 ? getPair(inKept(k, b, e, 0)) : next_c[e];
                if (RB == 1) xr[e] = next_r[e];
            }
            prefetch(k, b + kSmallWaves);
#pragma unroll
            for (int o = 0; o < RB; ++o) {
                f32x16 vc = zero16(), vr = zero16();
#pragma unroll
                for (int e = 0; e < RB; ++e) {
                    const Pair pe = operandP(o, e);
                    if (k)
                        multiplyBoth(pe, y[e], vc, vr);
                    else
                        vc = multiply(pe, y[e], vc);
                }
                vc *= f2.turn;
                vr *= f2.turn;
#pragma unroll
                for (int e = 0; e < RB; ++e) {
                    const Pair ne = RB == 1 ? own_n : readSymmetric<RB>(M, o, e, lane);
                    if (k)
                        multiplyBoth(ne, x[e], vc, vr);
                    else
                        vc = multiply(ne, x[e], vc);
                }
                vc *= f2.acc;
                if (k) {
                    Pair c;
                    c.set(vc);
                    putPair(inLds(b, o), c);  // (y has been read)
                    l[o].set(vr * f2.acc);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) dot += (double)vc[i] * (double)x[o].value(i);
                    putPair(inLds(b, o), __builtin_bit_cast(Pair, vc));  // Y_0 stays in float32
                }
            }
            if (k) {
                if (RB > 1) {
#pragma unroll
                    for (int e = 0; e < RB; ++e) xr[e] = getPair(inKept(k - 1, b, e, 1));
                }
                addBoth(l, xr);
            }
        }
    }
    // through X_0 = G / (|G| + eps), as in tail_kernel
    dot = blockSum(dot, sums);
    const double back = 1.0 / (norm.x_scale * norm.plus), ky = 1.0 / norm.plus;
    const double kx = norm.size > 0.0 ? dot * back / norm.size * back : norm.size;
#pragma unroll 1
    for (int b = wave; b < blocks; b += kSmallWaves) {
        const int j = b * 32 + (lane & 31);
#pragma unroll
        for (int p = 0; p < RB; ++p) {
            const Pair x = getPair(inKept(0, b, p, 0));
            const f32x16 y = __builtin_bit_cast(f32x16, getPair(inLds(b, p)));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = p * 32 + laneRow(i, lane);
                if (row < s && j < w)
                    global<T>(r.out)[row * r.out_rs + j * r.out_cs] =
                        fromFloat<T>((float)(ky * (double)y[i] - kx * (double)x.value(i)));
            }
        }
    }
}

// ---- the end of the gradient: through X_0 = G / (|G| + eps) ------------------------------------
//
//     dG = Y_0 / (|G| + eps) - X_0 <Y_0, X_0> / |G|
//
// Two passes, bound by HBM: of eight 1024^2 float32 matrices the dot products take 14 us (8 bytes an
// element, 4.8 TB/s), the result 21 us (12 bytes, 4.7 TB/s).

struct TailArgs {
    Shapes sh;
    const MatRec *recs;
    const MatNorm *norms;
    char *ws, *kept;
    double *parts;                              // <Y_0, X_0 * 2^e>, or <X, X>
    int64_t y[kMaxGroups], x[kMaxGroups];       // float rows of Y_0; X_0 or another operand
    int64_t per[kMaxGroups];                    // dot: cells of 32 x 32 per workgroup
    int nparts[kMaxGroups];
};

template <bool SQUARE> __global__ __launch_bounds__(256) void dot_kernel(TailArgs a) {
    __shared__ double lds[4];
    int part = blockIdx.x, mat;
    const int gi = findGroup(a.sh, part, mat);
    const Group &g = a.sh.g[gi];
    const Region region(a.ws, a.kept, g, mat);
    mat += g.mat0;
    const int64_t wp = padded(g.w), ld = rowBytes(wp, true);
    const int across = (int)(wp / 32);
    const int64_t cells = (int64_t)((g.s + 31) / 32) * across, from = part * a.per[gi];
    const int64_t to = from + a.per[gi] < cells ? from + a.per[gi] : cells;
    double sum = 0.0;
    // 128 chunks to a cell
    for (int64_t q = from * 128 + threadIdx.x; q < to * 128; q += 256) {
        const int64_t cell = q >> 7;
        const int i = (int)(cell / across) * 32 + (int)(q & 31);
        const int j = (int)(cell % across) * 32 + (int)(q >> 5 & 3) * 8;
        if (i >= g.s || j >= g.w) continue;
        float x[8], y[8];
        loadOperand(chunkOf(region + a.x[gi], ld, i, j, true), x);
        if (!SQUARE) load8((const float *)(region + a.y[gi]) + i * wp + j, g.w - j, y);
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += (double)x[k] * (double)(SQUARE ? x[k] : y[k]);
    }
    sum = blockSum(sum, lds);
    if (threadIdx.x == 0) a.parts[(int64_t)mat * kMaxParts + part] = sum;
}

template <typename T> __global__ __launch_bounds__(256) void tail_kernel(TailArgs a) {
    __shared__ float tile[64][65];
    __shared__ double lds[4];
    int t = blockIdx.x, mat;
    const int gi = findGroup(a.sh, t, mat);
    const Group &g = a.sh.g[gi];
    const Region region(a.ws, a.kept, g, mat);
    mat += g.mat0;
    const MatRec &r = a.recs[mat];
    const MatNorm n = a.norms[mat];
    const double dot = blockSum(
        (int)threadIdx.x < a.nparts[gi] ? a.parts[(int64_t)mat * kMaxParts + threadIdx.x] : 0.0, lds);
    const double back = 1.0 / (n.x_scale * n.plus);  // stored X_0 * back = X_0 (a power of two)
    const double ky = 1.0 / n.plus;
    const double kx = n.size > 0.0 ? dot * back / n.size * back : n.size;  // (NaN stays NaN)
    const int64_t wp = padded(g.w), ld = rowBytes(wp, true);
    const int across = (int)(wp / 64), i0 = t / across * 64, j0 = t % across * 64;
    for (int q = threadIdx.x; q < 512; q += 256) {
        const int i = i0 + (q >> 3), c = (q & 7) * 8, j = j0 + c;
        float x[8], y[8];
        if (i < g.s && j < g.w) {
            loadOperand(chunkOf(region + a.x[gi], ld, i, j, true), x);
            load8((const float *)(region + a.y[gi]) + i * wp + j, g.w - j, y);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                tile[q >> 3][c + k] = (float)(ky * (double)y[k] - kx * (double)x[k]);
        }
    }
    __syncthreads();
    const bool by_rows = r.out_cs <= r.out_rs;
    const int lane = threadIdx.x & 63;
    for (int q = threadIdx.x >> 6; q < 64; q += 4) {
        const int di = by_rows ? q : lane, dj = by_rows ? lane : q;
        if (i0 + di < g.s && j0 + dj < g.w)
            global<T>(r.out)[(i0 + di) * r.out_rs + (j0 + dj) * r.out_cs] = fromFloat<T>(tile[di][dj]);
    }
}

// ---- 8-bit blocks ------------------------------------------------------------------------------
//
// Bound by HBM: 67 million elements to codes and scales, 59 us from float32 = 5.8 TB/s, 46 us from 16-bit
// types = 4.4 (the arithmetic is the same for half the bytes); back 61 us = 5.5 TB/s and 31 us = 6.6.

constexpr int kListMax = 64;
struct BlocksArgs {
    int n;
    const void *in[kListMax];
    void *out[kListMax];
    float *scales[kListMax];
    size_t count[kListMax];
    unsigned tile0[kListMax];  // a workgroup takes 2048 elements
};

__device__ inline int findArray(const BlocksArgs &a, unsigned b) {
    int lo = 0, hi = a.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (b >= a.tile0[mid]) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <typename T> __global__ __launch_bounds__(256) void quantize_kernel(BlocksArgs a) {
    const int k = findArray(a, blockIdx.x);
    const int64_t n = (int64_t)a.count[k];
    const int64_t e = (int64_t)(blockIdx.x - a.tile0[k]) * 2048 + (int64_t)threadIdx.x * 8;
    const int valid = e >= n ? 0 : n - e < 8 ? (int)(n - e) : 8;
    float v[8];
    unsigned long long peak = 0;
    load8((const T *)a.in[k] + e, valid, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned long long m =
            (unsigned long long)__double_as_longlong((double)v[i]) & 0x7fffffffffffffffull;
        peak = m > peak ? m : peak;
    }
    const float scale = scaleOf(blockPeak(peak));
    const double reciprocal = 1.0 / (double)scale;
    int8_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = (int8_t)codeOf((double)v[i], scale, reciprocal);
    int8_t *o = (int8_t *)a.out[k] + e;
    if (valid == 8 && ((uintptr_t)o & 7) == 0) {
        *global<int64_t>((void *)o) = pack8(c);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) global<int8_t>((void *)o)[i] = c[i];
    }
    if (valid && (e & 127) == 0) global<float>((void *)a.scales[k])[e >> 7] = scale;
}

template <typename T> __global__ __launch_bounds__(256) void dequantize_kernel(BlocksArgs a) {
    const int k = findArray(a, blockIdx.x);
    const int64_t n = (int64_t)a.count[k];
    const int64_t e = (int64_t)(blockIdx.x - a.tile0[k]) * 2048 + (int64_t)threadIdx.x * 8;
    if (e >= n) return;
    const int valid = n - e < 8 ? (int)(n - e) : 8;
    const int8_t *p = (const int8_t *)a.in[k] + e;
    const float scale = global<float>(a.scales[k])[e >> 7];
    int8_t c[8];
    if (valid == 8 && ((uintptr_t)p & 7) == 0) {
        unpack8(*global<int64_t>(p), c);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = i < valid ? global<int8_t>(p)[i] : (int8_t)0;
    }
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)c[i] * scale;
    store8((T *)a.out[k] + e, valid, v);
}

}  // namespace toa_muon
