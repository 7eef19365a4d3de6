// Host side of libtoa_muon.so (include/toa_muon.h): checks, the plan of a list (matrices sorted by
// shape, in batches that a workspace of bounded size holds), and the launches.  Everything a kernel
// reads beside the caller's tensors travels in launch arguments or is made on the device, so a call
// allocates nothing and leaves nothing behind.
#include <algorithm>
#include <cmath>
#include <limits>
#include <vector>

#include "muon_kernels.hpp"
#include "toa_muon.h"

using namespace toa_muon;

namespace {

// A batch's regions stay below this (one matrix alone may be larger).  Large batches fill whole
// rounds of tiles: 96 matrices of 1024^2 take 7.2 ms in one batch and 8.0 in three, GPT-2-medium's 144
// matrices (bfloat16 step) 16.4 ms in two batches, 17.6 in 1 GiB and 21.4 in 256 MiB, which stay in the
// last-level cache.  (One of 8 GiB and two of 4 take the same, side by side: 15.9.)
constexpr int64_t kBatchBytes = (int64_t)4 << 30;
constexpr int kBatchMats = 4096;
constexpr int64_t kMaxDim = (int64_t)1 << 20;

int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// What a plan is for.  Keep: the forward pass leaves its iterates in a buffer of the caller's, and the
// gradient (kGradientKept) finds them there.
enum Purpose { kForward, kForwardKeep, kGradient, kGradientKept };

// Where one matrix's buffers lie: offsets into its region, or into the kept iterates.
struct Layout {
    int64_t x[kMaxSteps + 1], xt[kMaxSteps + 1], s[kMaxSteps], p[kMaxSteps];  // (gradient: step by step)
    int64_t t, y[2], yt[2], m, n, yf, bytes, kept_bytes;
};

Layout layoutOf(int s, int w, int steps, Purpose purpose) {
    Layout l{};
    auto take = [&](int64_t &at, int64_t rows, int64_t cols) {
        const int64_t here = at;
        at += align256((rows + kRows - 1) / kRows * kRows * rowBytes(padded(cols), true));
        return here;
    };
    int64_t at = 0;
    if (purpose != kForward) {
        // every iterate is kept: the way back needs them in reverse
        const int64_t where = purpose == kGradient ? 0 : kKept;
        for (int k = 0; k < steps; ++k) {
            l.x[k] = take(at, s, w) | where;
            l.xt[k] = take(at, w, s) | where;
            l.s[k] = take(at, s, s) | where;
            l.p[k] = take(at, s, s) | where;
        }
        if (where) std::swap(at, l.kept_bytes);
        if (purpose != kForwardKeep) {
            for (int k = 0; k < 2; ++k) {
                l.y[k] = take(at, s, w);
                l.yt[k] = take(at, w, s);
            }
            l.m = take(at, s, s);
            l.n = take(at, s, s);
            l.yf = take(at, s, w);
        }
    } else {
        const int64_t x0 = take(at, s, w), x0t = take(at, w, s);
        const int64_t x1 = steps > 1 ? take(at, s, w) : 0, x1t = steps > 1 ? take(at, w, s) : 0;
        const int64_t ss = take(at, s, s), pp = take(at, s, s);
        l.t = take(at, s, s);
        for (int k = 0; k <= steps; ++k) {
            l.x[k] = k & 1 ? x1 : x0;
            l.xt[k] = k & 1 ? x1t : x0t;
        }
        for (int k = 0; k < steps; ++k) {
            l.s[k] = ss;
            l.p[k] = pp;
        }
    }
    l.bytes = at;
    return l;
}

struct Batch {
    std::vector<size_t> mats;  // indices into the caller's list, shape by shape
    struct Shape {
        int s, w, mat0, count;
        int64_t base, kept_base;
        Layout lay;
    };
    std::vector<Shape> shapes;
    int64_t bytes = 0;  // of all regions
};

// Head of the workspace: records, norms, partial sums (two sets) and factors of a batch.
struct Head {
    int64_t recs, norms, parts, parts_y, factors, regions;
};

int stagesOf(int steps, bool backward) { return (kStepFactors + (backward ? 3 : 0)) * steps; }

Head headOf(int64_t mats, int stages) {
    Head h;
    h.recs = 0;
    h.norms = align256(mats * (int64_t)sizeof(MatRec));
    h.parts = h.norms + align256(mats * (int64_t)sizeof(MatNorm));
    h.parts_y = h.parts + align256(mats * kMaxParts * 8);
    h.factors = h.parts_y + align256(mats * kMaxParts * 8);
    h.regions = h.factors + align256(mats * stages * (int64_t)sizeof(Factor));
    return h;
}

// Small matrices (see small_kernel): those of one kernel variant, `stride` bytes of kept iterates
// for each in the gradient.
struct SmallBatch {
    int rb;
    std::vector<size_t> mats;
    int64_t stride = 0;

    // records (where they do not fit in the launch), then the kept iterates
    int64_t records() const {
        return mats.size() > kSmallInline ? align256((int64_t)mats.size() * (int64_t)sizeof(MatRec)) : 0;
    }
    int64_t bytes() const { return records() + (int64_t)mats.size() * stride; }
};

// The way back bounds each cotangent by the one before.  Bounds that run ahead of the truth cost the
// operands their low bits, so where a bound may have grown by more than this the norm is measured anew
// (the default coefficients: 394 at their five steps, so never there).
constexpr double kMaxGrowth = 512.0;

// Tiles of 64 x 64 that small matrices may add to the launches of larger ones (which hold 512 at once).
constexpr int64_t kFewTiles = 128;

// Rows / 32 of the variant that takes an s x w matrix, or 0: what its LDS holds.  The one for 64 rows spills
// 55 to 65 registers, and is ahead of the tiles or level with them all the same: one 64 x 64 float32 matrix 52
// us (77), its gradient 154 (193); one 33 x 224 62 (64) and 189 (200), one 64 x 224 64 (63) and 198 (197); 256
// of these 94 (124) and 313 (431).
int smallVariant(int64_t s, int64_t w) {
    for (int rb = 1; rb <= 2; ++rb)
        if (s <= 32 * rb) return w <= 32 * smallColumnBlocks(rb) ? rb : 0;
    return 0;
}

// `bytes`: of the workspace; `kept`: of the kept iterates, which lie in the order of the sorted list and
// so do not depend on how it falls into batches.
int plan(size_t num, const int64_t *rows, const int64_t *cols, const Series &series, Purpose purpose,
         std::vector<Batch> &batches, std::vector<SmallBatch> &smalls, int64_t &bytes, int64_t &kept_bytes) {
    const bool backward = purpose == kGradient || purpose == kGradientKept;
    const int steps = series.steps;
    // (small_kernel measures nothing on its way back)
    double growth = 1.0;
    for (int k = 1; k < steps; ++k) growth *= series.d[k];
    const bool small = purpose == kForward || growth <= kMaxGrowth;
    bytes = kept_bytes = 0;
    auto key = [&](size_t i) {
        return std::make_pair(std::min(rows[i], cols[i]), std::max(rows[i], cols[i]));
    };
    std::vector<size_t> order, few;  // through the tiles; small ones
    order.reserve(num);
    int64_t few_tiles = 0;
    for (size_t i = 0; i < num; ++i) {
        if (rows[i] < 0 || cols[i] < 0 || rows[i] > kMaxDim || cols[i] > kMaxDim) return TOA_ESIZE;
        if (!rows[i] || !cols[i]) continue;
        const auto shape = key(i);
        if (small && smallVariant(shape.first, shape.second)) {
            few.push_back(i);
            few_tiles += (shape.first + 63) / 64 * ((shape.second + 63) / 64);
        } else {
            order.push_back(i);
        }
    }
    // A few small ones beside larger ones go with them: their tiles find room in launches that are made
    // anyway, which costs next to nothing, and a launch of their own 20 to 50 us.
    if (!order.empty() && few_tiles <= kFewTiles) {
        std::vector<std::pair<int64_t, int64_t>> shapes;
        for (const auto *list : {&order, &few})
            for (size_t i : *list) shapes.push_back(key(i));
        std::sort(shapes.begin(), shapes.end());
        if (std::unique(shapes.begin(), shapes.end()) - shapes.begin() <= kMaxGroups) {
            order.insert(order.end(), few.begin(), few.end());
            few.clear();
        }
    }
    for (size_t i : few) {
        const auto shape = key(i);
        const int rb = smallVariant(shape.first, shape.second);
        const int64_t kept = backward ? align256(steps * smallKept(rb, (int)shape.second)) : 0;
        auto it = std::find_if(smalls.rbegin(), smalls.rend(),
                               [&](const SmallBatch &b) { return b.rb == rb; });
        SmallBatch *b = it == smalls.rend() ? nullptr : &*it;
        if (!b || ((int64_t)b->mats.size() + 1) * std::max(b->stride, kept) > kBatchBytes) {
            smalls.push_back({rb, {}, 0});
            b = &smalls.back();
        }
        b->mats.push_back(i);
        b->stride = std::max(b->stride, kept);
    }
    for (const SmallBatch &b : smalls) bytes = std::max(bytes, b.bytes());
    // (long rows first: their tiles take longest and should not be what a launch ends with)
    std::stable_sort(order.begin(), order.end(), [&](size_t i, size_t j) {
        return std::make_pair(key(i).second, key(i).first) > std::make_pair(key(j).second, key(j).first);
    });
    Layout lay{};
    for (size_t k = 0; k < order.size(); ++k) {
        const auto shape = key(order[k]);
        const bool same = k && shape == key(order[k - 1]);
        if (!same) lay = layoutOf((int)shape.first, (int)shape.second, steps, purpose);
        Batch *b = batches.empty() ? nullptr : &batches.back();
        if (!b || b->bytes + lay.bytes > kBatchBytes || (int)b->mats.size() == kBatchMats ||
            (!same && (int)b->shapes.size() == kMaxGroups)) {
            batches.emplace_back();
            b = &batches.back();
        }
        if (b->shapes.empty() || !same)
            b->shapes.push_back({(int)shape.first, (int)shape.second, (int)b->mats.size(), 0,
                                 b->bytes, kept_bytes, lay});
        b->shapes.back().count++;
        b->mats.push_back(order[k]);
        b->bytes += lay.bytes;
        kept_bytes += lay.kept_bytes;
    }
    for (const Batch &b : batches)
        bytes = std::max(bytes, headOf((int64_t)b.mats.size(), stagesOf(steps, backward)).regions + b.bytes);
    return 0;
}

// The largest |f| on [0, top] of f(t) = k0 t^n0 + k1 t^(n0+2) + k2 t^(n0+4), n0 = 0 or 1.
double largest(double k0, double k1, double k2, int n0, double top) {
    auto at = [&](double t) {
        const double q = t * t;
        return std::fabs((k0 + q * (k1 + q * k2)) * (n0 ? t : 1.0));
    };
    double best = std::max(at(0.0), at(top));
    // zeros of the derivative, a quadratic (n0 = 1) or linear (n0 = 0) equation in q = t^2
    auto consider = [&](double q) {
        if (q > 0.0 && q < top * top) best = std::max(best, at(std::sqrt(q)));
    };
    if (n0) {
        const double qa = 5.0 * k2, qb = 3.0 * k1, qc = k0;
        if (qa == 0.0) {
            if (qb != 0.0) consider(-qc / qb);
        } else {
            const double disc = qb * qb - 4.0 * qa * qc;
            if (disc >= 0.0) {
                consider((-qb + std::sqrt(disc)) / (2.0 * qa));
                consider((-qb - std::sqrt(disc)) / (2.0 * qa));
            }
        }
    } else if (k2 != 0.0) {
        consider(-k1 / (2.0 * k2));
    }
    return best;
}

// The smallest |a + b q + c q^2| on [0, top].
double smallest(double a, double b, double c, double top) {
    auto at = [&](double q) { return a + q * (b + q * c); };
    double lo = std::min(at(0.0), at(top)), hi = std::max(at(0.0), at(top));
    if (c != 0.0) {
        const double q = -b / (2.0 * c);
        if (q > 0.0 && q < top) {
            lo = std::min(lo, at(q));
            hi = std::max(hi, at(q));
        }
    }
    return lo > 0.0 ? lo : hi < 0.0 ? -hi : 0.0;
}

int checkSeries(const toa_muon_series *q) {
    if (!q) return TOA_ENULL;
    if (q->steps < 1 || q->steps > kMaxSteps || !std::isfinite(q->a) || !std::isfinite(q->b) ||
        !std::isfinite(q->c) || !(q->eps >= 0.0) || !std::isfinite(q->eps))
        return TOA_EVALUE;
    return 0;
}

// Bounds of the iterates from a start of norm 1 (with a hundredth of slack for rounding).  An iterate that
// may stay far below its bound loses its low bits (beyond 2^18 columns even at 64), so series that may
// grow further before their last step are refused.
int boundsOf(const toa_muon_series &q, Series &f) {
    f.a = (float)q.a;
    f.b = (float)q.b;
    f.c = (float)q.c;
    f.eps = q.eps;
    f.steps = q.steps;
    double x = 1.0;
    for (int k = 0; k <= q.steps; ++k) {
        f.x[k] = 1.01 * x;
        if (k == q.steps) break;
        f.r[k] = std::max(1.01 * largest(q.a, q.b, q.c, 0, f.x[k]), 1e-3);
        f.d[k] = std::max(1.01 * largest(q.a, 3.0 * q.b, 5.0 * q.c, 0, f.x[k]), 1e-3);
        // (operands are scaled by 2^-110 at most)
        if (!(std::max(f.r[k], f.d[k]) <= 1e30)) return TOA_EVALUE;
        x = std::max(largest(q.a, q.b, q.c, 1, f.x[k]), 1e-6);
        if (k + 1 < q.steps && !(x <= 64.0)) return TOA_EVALUE;
    }
    // completing the square takes c h^2 away from what (X X^T + h I)^2 brings in: a bit of a or so
    // at most
    f.h = q.c != 0.0 ? q.b / (2.0 * q.c) : 0.0;
    f.square = q.c != 0.0 && std::fabs(q.c) * f.h * f.h <= 2.0 * std::fabs(q.a);
    // What is off in the multiple of I in P is off everywhere, and in every step: where S is small beside it
    // (few large singular values) it is most of the error.  So h is a number that an operand holds exactly,
    // and the multiple of I that P is given takes what the product makes of it -- with c as a float, and
    // without the square of h's low half -- to a.  (a - b h / 2, with h and b each rounded by itself: 1.3e-6
    // off in gradients of rank one, now 7e-7; 100 x 100 of full rank 1.1e-6, now 9e-7.)
    f.unit = q.a;
    if (f.square) {
        auto half = [](double v) {
            int e;
            const double m = std::frexp(v, &e);
            return std::ldexp(std::nearbyint(std::ldexp(m, 11)), e - 11);
        };
        const double exact = (float)f.h, hi = half(exact), lo = half(exact - hi);
        f.h = hi + lo;
        f.unit = q.a - (double)f.c * (f.h * f.h - lo * lo);
    }
    // Operands of 11 bits in the last step, each element off by 2^-12 of itself: that of X moves the
    // result by the slope, that of S (or S + h I, as it is kept) by what P changes with it, that of P by P
    // itself, all beside a result of |P X| >= (least |P|) |X|.  Up to 8 times 2^-12 is half a step of
    // bfloat16.  (The default coefficients reach 21, as c h^2 cancels most of a: with two such steps few
    // large singular values came out up to 2.6 roundings off.  Those that converge, (1.875, -1.25, 0.375)
    // or (2, -1.5, 0.5), take 6: five steps of 4 matrices of 4096 x 1024 in 765 us, at 22 bits throughout
    // 880; of 24 of 1024^2 in 1.68 ms, 1.88.)
    const double top = f.x[q.steps - 1] * f.x[q.steps - 1];
    const double kept = f.square ? std::max(std::fabs(f.h), std::fabs(f.h + top)) : top;
    const double of_s = f.square ? 2.0 * std::fabs(q.c) * kept
                                 : std::max(std::fabs(q.b), std::fabs(q.b + 2.0 * q.c * top));
    f.halves = f.d[q.steps - 1] + of_s * kept + f.r[q.steps - 1] <= 8.0 * smallest(q.a, q.b, q.c, top);
    return 0;
}

template <typename... Args>
int launch(void (*kernel)(Args...), int64_t grid, int block, hipStream_t stream, Args... args) {
    if (grid <= 0) return 0;
    if (grid > std::numeric_limits<int>::max()) return TOA_ESIZE;
    void *ptrs[] = {(void *)&args...};
    return (int)hipLaunchKernel((const void *)kernel, dim3((unsigned)grid), dim3(block), ptrs, 0,
                                stream);
}

#define TRY(expr)                   \
    do {                            \
        const int rc_ = (expr);     \
        if (rc_ != 0) return rc_;   \
    } while (0)

// fn(element type) for a dtype code.
template <typename F> int withType(int dtype, F fn) {
    switch (dtype) {
        case TOA_F32: return fn(float());
        case TOA_F16: return fn(_Float16());
        case TOA_BF16: return fn(__bf16());
        default: return TOA_EDTYPE;
    }
}

enum What { kOrthogonalize, kStep, kBackward };

struct Call {
    What what;
    int dtype, momentum_dtype;
    const int64_t *rows, *cols;
    const toa_muon_view *g, *aux, *out;  // aux: momentum or cotangent
    float *const *scales;
    const toa_muon_hyper *hyper;
    toa_muon_series series;
    char *ws, *kept;  // kept: or null
    hipStream_t stream;
};

double shapeRate(int adjust, int64_t rows, int64_t cols) {
    if (adjust == TOA_MUON_ASPECT) return std::sqrt(std::max(1.0, (double)rows / (double)cols));
    if (adjust == TOA_MUON_RMS) return 0.2 * std::sqrt((double)std::max(rows, cols));
    return 1.0;
}

MatRec recordOf(const Call &c, size_t i) {
    const bool turned = c.rows[i] > c.cols[i];
    MatRec r{};
    auto put = [&](const toa_muon_view &v, int64_t &rs, int64_t &cs) {
        rs = turned ? v.col_stride : v.row_stride;
        cs = turned ? v.row_stride : v.col_stride;
        return v.data;
    };
    r.g = put(c.g[i], r.g_rs, r.g_cs);
    r.out = put(c.out[i], r.out_rs, r.out_cs);
    if (c.aux) r.aux = put(c.aux[i], r.aux_rs, r.aux_cs);
    r.scales = c.scales ? c.scales[i] : nullptr;
    r.rate = 1.f;
    if (c.hyper) {
        const double rate = shapeRate(c.hyper->adjust, c.rows[i], c.cols[i]);
        r.rate = (float)(c.hyper->apply ? c.hyper->lr * rate : rate);
        r.keep = (float)(1.0 - c.hyper->lr * c.hyper->weight_decay);
    }
    r.s = (int)std::min(c.rows[i], c.cols[i]);
    r.w = (int)std::max(c.rows[i], c.cols[i]);
    return r;
}

int fillRecords(const Call &c, const std::vector<size_t> &mats, MatRec *to) {
    for (size_t from = 0; from < mats.size(); from += kFill) {
        FillArgs a{};
        const int n = (int)std::min<size_t>(kFill, mats.size() - from);
        for (int k = 0; k < n; ++k) a.r[k] = recordOf(c, mats[from + k]);
        TRY(launch(fill_kernel, 1, 64, c.stream, a, to + from, n));
    }
    return 0;
}

StepArgs stepOf(const Call &c) {
    if (!c.hyper) return StepArgs{};
    return {c.hyper->momentum, c.hyper->maximize ? -1.f : 1.f, c.hyper->nesterov};
}

template <typename T, int RB> auto smallKernel(const Call &c) {
    if (c.what == kBackward) return small_kernel<T, kPackG, RB, true>;
    if (c.what == kOrthogonalize) return small_kernel<T, kPackG, RB, false>;
    return c.momentum_dtype == TOA_I8      ? small_kernel<T, kPackMI8, RB, false>
           : c.momentum_dtype == c.dtype ? small_kernel<T, kPackM, RB, false>
                                          : small_kernel<T, kPackMF32, RB, false>;
}

int runSmall(const Call &c, const SmallBatch &b, const Series &series) {
    SmallArgs a{};
    a.q = series;
    // float32: S without h I, whose rounding is a good part of what a sum over few columns is off by
    // (16 x 16: 1.6e-6 with it, 6e-7 without and with all partial products, plain float32 8e-7; 22 -> 24
    // us for three of 32 x 288, their gradient 78 -> 85)
    if (c.dtype == TOA_F32) {
        a.q.square = 0;
        a.q.unit = c.series.a;
    }
    a.step = stepOf(c);
    a.apply = c.hyper && c.hyper->apply;
    a.stride = b.stride;
    a.ws = c.ws + b.records();
    if (b.records()) {
        a.recs = (const MatRec *)c.ws;
        TRY(fillRecords(c, b.mats, (MatRec *)c.ws));
    } else {
        for (size_t k = 0; k < b.mats.size(); ++k) a.r[k] = recordOf(c, b.mats[k]);
    }
    return withType(c.dtype, [&](auto t) {
        using T = decltype(t);
        return launch(b.rb == 1 ? smallKernel<T, 1>(c) : smallKernel<T, 2>(c),
                      (int64_t)b.mats.size(), kSmallWaves * 64, c.stream, a);
    });
}

class Run {
  public:
    Run(const Call &c, const Batch &b, const Series &series)
        : c_(c), b_(b), steps_(c.series.steps), back_(c.what == kBackward),
          keep_(c.kept != nullptr), few_(b.mats.size() <= kFew), stages_(stagesOf(steps_, back_)), head_(headOf((int64_t)b.mats.size(), stages_)),
          f_{series} {
        f_.q.paired = pairedSteps();
    }

    int go() {
        if (!few_) TRY(fillRecords(c_, b_.mats, (MatRec *)(c_.ws + head_.recs)));
        TRY(sums());
        TRY(factors());
        if (!back_ || !keep_) {
            TRY(pack(false, few_));
            int from = 0;  // which of the two buffers holds X
            for (int k = 0; k < f_.q.paired; k += 2, from ^= 1) TRY(forwardPair(k, from));
            for (int k = f_.q.paired; k < steps_; ++k, from ^= 1)
                TRY(forwardStep(k, back_ || keep_ ? k : from));
        }
        if (!back_) return 0;
        TRY(pack(true, few_ && keep_));
        double growth = 1.0;
        for (int k = steps_ - 1; k >= 0; --k) {
            if (k && k + 1 < steps_ && growth * f_.q.d[k] > kMaxGrowth) {
                TRY(measure(k + 1));
                growth = 1.0;
            }
            growth *= f_.q.d[k];
            TRY(backwardStep(k));
        }
        return dots<false>(0);
    }

  private:
    // whether step k's operands carry 22 bits (see boundsOf)
    bool split(int k) const {
        return back_ || keep_ || c_.dtype != TOA_BF16 || !f_.q.halves || k < f_.q.paired || k < steps_ - 1;
    }

    // Steps taken by twos: where that is less work for the batch (see muon_kernels.hpp).
    int pairedSteps() const {
        double one = 0.0, two = 0.0;  // of two steps
        for (const auto &s : b_.shapes) {
            const double n = (double)s.count * s.s * s.s;
            one += n * (6.0 * s.w + 2.0 * s.s);
            two += n * (3.0 * s.w + 5.0 * s.s);
        }
        return !back_ && !keep_ && two < 0.95 * one ? steps_ / 2 * 2 : 0;
    }

    const MatRec *recs() const { return (const MatRec *)(c_.ws + head_.recs); }

    // Shapes of a launch with tilesOf(shape) workgroups for each matrix.
    template <typename F> int64_t shapes(Shapes &sh, F tilesOf) const {
        int64_t at = 0;
        sh.n = (int)b_.shapes.size();
        for (int k = 0; k < sh.n; ++k) {
            const auto &s = b_.shapes[k];
            const int64_t tiles = tilesOf(s, k);
            sh.g[k] = {head_.regions + s.base, s.lay.bytes, s.kept_base, s.lay.kept_bytes,
                       s.s, s.w, s.mat0,
                       (int)at, (int)tiles, (int)(tiles * s.count)};
            at += tiles * s.count;
            if (at > std::numeric_limits<int>::max()) return at;
        }
        return at;
    }

    int sums() {
        SumArgs a{};
        a.recs = recs();
        a.parts = (double *)(c_.ws + head_.parts);
        a.step = stepOf(c_);
        if (few_) {
            a.few = (int)b_.mats.size();
            for (int k = 0; k < a.few; ++k) a.r[k] = recordOf(c_, b_.mats[k]);
        }
        const int64_t grid = shapes(a.sh, [&](const Batch::Shape &s, int k) {
            const int64_t n = (int64_t)s.s * s.w;
            // (at least eight elements a thread: more in a row, with few of them at work, cost a
            // list of odd small matrices 10 us)
            int64_t per = std::max<int64_t>(2048, (n + kMaxParts - 1) / kMaxParts);
            per = (per + 2047) / 2048 * 2048;
            a.per[k] = per;
            f_.nparts[k] = (int)((n + per - 1) / per);
            f_.mat_end[k] = s.mat0 + s.count;
            return (int64_t)f_.nparts[k];
        });
        f_.ngroups = a.sh.n;
        return withType(c_.dtype, [&](auto t) {
            using T = decltype(t);
            if (c_.what != kStep) {
                TRY(launch(sum_kernel<T, kSumG>, grid, 256, c_.stream, a));
                if (!back_) return 0;
                a.parts = (double *)(c_.ws + head_.parts_y);
                return launch(sum_kernel<T, kSumAux>, grid, 256, c_.stream, a);
            }
            return launch(c_.momentum_dtype == TOA_I8      ? sum_kernel<T, kMomentumI8>
                          : c_.momentum_dtype == c_.dtype ? sum_kernel<T, kMomentum>
                                                           : sum_kernel<T, kMomentumF32>,
                          grid, 256, c_.stream, a);
        });
    }

    int factors() {
        f_.parts = (const double *)(c_.ws + head_.parts);
        f_.parts_y = back_ ? (const double *)(c_.ws + head_.parts_y) : nullptr;
        f_.norms = (MatNorm *)(c_.ws + head_.norms);
        f_.factors = (Factor *)(c_.ws + head_.factors);
        f_.stages = stages_;
        f_.measured = -1;
        return few_ ? 0 : launch(factors_kernel, (int64_t)b_.mats.size(), 256, c_.stream, f_);
    }

    // The cotangent, or the matrix itself, as operands.
    int pack(bool cotangent, bool with_factors) {
        return with_factors ? pack<true>(cotangent) : pack<false>(cotangent);
    }

    template <bool FEW> int pack(bool cotangent) {
        PackArgs a{};
        a.f = f_;
        a.recs = recs();
        a.norms = (const MatNorm *)(c_.ws + head_.norms);
        a.ws = c_.ws;
        a.kept = c_.kept;
        a.split = split(0);
        a.step = stepOf(c_);
        const int64_t grid = shapes(a.sh, [&](const Batch::Shape &s, int k) {
            a.off[k] = cotangent ? s.lay.y[0] : s.lay.x[0];
            a.off_t[k] = cotangent ? s.lay.yt[0] : s.lay.xt[0];
            return padded(s.s) / 64 * (padded(s.w) / 64);
        });
        return withType(c_.dtype, [&](auto t) {
            using T = decltype(t);
            return launch(cotangent                          ? pack_kernel<T, kPackAux, FEW>
                          : c_.what != kStep               ? pack_kernel<T, kPackG, FEW>
                          : c_.momentum_dtype == TOA_I8    ? pack_kernel<T, kPackMI8, FEW>
                          : c_.momentum_dtype == c_.dtype ? pack_kernel<T, kPackM, FEW>
                                                           : pack_kernel<T, kPackMF32, FEW>,
                          grid, 256, c_.stream, a);
        });
    }

    // One launch of the product for every matrix of the batch.  `operands` names a matrix's
    // buffers; steps1 = 1 there says that there is a second pair.
    template <typename F>
    int product(int stage, int k, bool split_out, bool symmetric, int mode, F operands) {
        GemmArgs a{};
        a.ws = c_.ws;
        a.kept = c_.kept;
        a.recs = recs();
        a.factors = (const Factor *)(c_.ws + head_.factors);
        a.stages = stages_;
        a.stage = stage;
        a.symmetric = symmetric;
        a.mode = mode;
        a.split_out = split_out;
        const bool sp = split(k);
        for (int g = 0; g < (int)b_.shapes.size(); ++g) {
            const Batch::Shape &s = b_.shapes[g];
            Product &p = a.p[g];
            p.e = p.d = p.dt = -1;
            const int ld_s = (int)rowBytes(padded(s.s), sp), ld_w = (int)rowBytes(padded(s.w), sp);
            operands(p, s.lay, ld_s, ld_w);
            p.rows = s.s;
            p.cols = symmetric ? s.s : s.w;
            p.lde = symmetric ? ld_s : ld_w;
            p.ldd = mode == kToFloat ? (int)padded(s.w) * 4
                                     : (int)rowBytes(padded(symmetric ? s.s : s.w), split_out);
            p.lddt = (int)rowBytes(padded(s.s), split_out);
            p.steps0 = p.lda / kPiece;
            if (p.steps1) p.steps1 = p.steps0;
        }
        const bool tensor = mode == kToTensor || mode == kToParam;
        return withType(tensor ? c_.dtype : TOA_F32, [&](auto t) {
            using T = decltype(t);
            switch (pickTiles(a, sp)) {
                case kTiles256:
                    return sp ? tiles<T, 256, 2, 4, 1, 2, true>(a) : tiles<T, 256, 2, 4, 1, 2, false>(a);
                case kTiles128Pair:
                    return sp ? tiles<T, 128, 2, 2, 1, 2, true>(a) : tiles<T, 128, 2, 2, 1, 2, false>(a);
                case kTiles128:
                    return sp ? tiles<T, 128, 2, 4, 1, 4, true>(a) : tiles<T, 128, 2, 4, 1, 4, false>(a);
                default:
                    return sp ? tiles<T, 64, 1, 1, 4, 2, true>(a) : tiles<T, 64, 1, 1, 4, 2, false>(a);
            }
        });
    }

    static int64_t tilesOf(const Product &p, bool symmetric, int size) {
        const int64_t tm = (p.rows + size - 1) / size, tn = (p.cols + size - 1) / size;
        return symmetric ? tm * (tm + 1) / 2 : tm * tn;
    }

    enum { kTiles256, kTiles128Pair, kTiles128, kTiles64, kVariants };

    // The variant that finishes first.  A tile's time is its start and stores plus its pieces: `alone`
    // on an empty chip, `full` where as many as fit are at work.  What is left after whole rounds
    // takes between the two: the large tiles as the square of the share filled; the 128 x 128 of which
    // two fit on a compute unit little more than one alone up to one to a unit, and most of a round
    // beyond; the 64 x 64 follow each other without rounds.
    // Microseconds of whole launches -- so with their start, the change of workgroups and the last to end --
    // fitted to 1..48 matrices of 1024^2, 2048^2, 4096^2, 16 x 512^2 and 64 x 256^2, to
    // 3..10 % (the 64 x 64 then 8 % up: long lists of different operands miss the L2 more); the variant
    // chosen is 0.3 % from the best of the four on average, 7 % at most.  Large
    // tiles get most out of a full chip (P X of 48 matrices of 1024^2: 324 us in 256 x 256, 379, 400
    // and 436 in 64 x 64), small ones start and end sooner and spread few results over more of it (of
    // one matrix: 65, 29, 26 and 13 us).
    int pickTiles(const GemmArgs &a, bool split_in) const {
        struct Variant {
            int size, at_once;  // tiles that the whole chip holds
            double alone, alone_piece, full, full_piece;
        };
        // with 22-bit operands, and with halves
        static const Variant table[2][kVariants] = {
            {{256, 256, 12.5, 1.67, 46.4, 2.18},
             {128, 512, 7.8, 0.66, 25.7, 1.24},
             {128, 256, 5.1, 0.63, 11.6, 0.70},
             {64, 512, 4.7, 0.21, 1.9, 0.54}},
            {{256, 256, 12.7, 1.26, 29.0, 1.54},
             {128, 512, 7.3, 0.63, 17.2, 0.97},
             {128, 256, 6.2, 0.50, 8.4, 0.58},
             {64, 512, 5.0, 0.26, 4.1, 0.42}}};
        const Variant *variants = table[!split_in];
        int best = 0;
        double least = 0.0;
        for (int k = 0; k < kVariants; ++k) {
            const Variant &v = variants[k];
            double tiles = 0.0, pieces = 0.0;
            for (int g = 0; g < (int)b_.shapes.size(); ++g) {
                const double n = (double)tilesOf(a.p[g], a.symmetric, v.size) * b_.shapes[g].count;
                tiles += n;
                pieces += n * (a.p[g].steps0 + a.p[g].steps1);
            }
            pieces /= tiles;
            const double alone = v.alone + v.alone_piece * pieces, full = v.full + v.full_piece * pieces;
            const double rounds = std::floor(tiles / v.at_once), rest = tiles / v.at_once - rounds;
            double time;
            if (k == kTiles64) {
                time = std::max(alone, v.alone + full * tiles / v.at_once);
            } else {
                const double share = k != kTiles128Pair ? rest * rest
                                     : rest <= 0.5      ? 0.3 * rest
                                                        : 0.4 + 0.6 * rest;
                const double more = std::max(0.0, full - alone);
                time = rounds * (alone + more) + (rest > 0.0 ? alone + more * share : 0.0);
            }
            if (k == 0 || time < least) {
                least = time;
                best = k;
            }
        }
        return best;
    }

    template <typename T, int B, int WM, int WN, int KS, int STAGES, bool SPLIT>
    int tiles(GemmArgs &a) {
        const int64_t grid = shapes(a.sh, [&](const Batch::Shape &, int g) {
            return tilesOf(a.p[g], a.symmetric, B);
        });
        return launch(gemm_kernel<T, B, B, WM, WN, KS, STAGES, SPLIT>, grid, WM * WN * KS * 64,
                      c_.stream, a);
    }

    // How the last product leaves.
    int lastMode() const { return c_.hyper && c_.hyper->apply ? kToParam : kToTensor; }

    // X' (or X'') = by(layout) X, from one buffer of X to another.
    template <typename F> int advance(int stage, int k, int next, int from, int to, F by) {
        const bool last = next == steps_;
        return product(stage, k, last || split(next), false, last ? lastMode() : kToOperand,
                       [&](Product &p, const Layout &l, int ld_s, int) {
                           p.a0 = by(l);
                           p.b0 = l.xt[from];
                           p.lda = p.ldb = ld_s;
                           if (!last) {
                               p.d = l.x[to];
                               p.dt = l.xt[to];
                           }
                       });
    }

    // A product of symmetric matrices that is symmetric itself.
    template <typename F> int symmetric(int stage, int k, F operands) {
        return product(stage, k, split(k), true, kToOperand,
                       [&](Product &p, const Layout &l, int ld_s, int) {
                           p.lda = p.ldb = ld_s;
                           operands(p, l);
                           p.dt = p.d;
                       });
    }

    int gram(int stage, int k, int from) {
        return product(stage, k, split(k), true, kToOperand,
                       [&](Product &p, const Layout &l, int, int ld_w) {
                           p.a0 = p.b0 = l.x[from];
                           p.lda = p.ldb = ld_w;
                           p.d = p.dt = l.s[k];
                       });
    }

    int forwardStep(int k, int from) {
        const int stage = kStepFactors * k;
        TRY(gram(stage, k, from));
        TRY(symmetric(stage + 1, k, [&](Product &p, const Layout &l) {
            p.a0 = p.b0 = l.s[k];
            if (!f_.q.square) p.e = l.s[k];
            p.d = l.p[k];
        }));
        if (back_ && k + 1 == steps_) return 0;  // the result itself is not needed
        return advance(stage + 2, k, k + 1, from, back_ || keep_ ? k + 1 : from ^ 1,
                       [&](const Layout &l) { return l.p[k]; });
    }

    // Two steps (S, P, T, S', P', Q, X''); S' takes S's place, P' T's, and Q that of S'.
    int forwardPair(int k, int from) {
        const int stage = kStepFactors * k;
        TRY(gram(stage, k, from));
        if (thin()) {
            TRY(squares(stage, k));
            return advance(stage + 6, k, k + 2, from, from ^ 1, [&](const Layout &l) { return l.s[k]; });
        }
        TRY(symmetric(stage + 1, k, [&](Product &p, const Layout &l) {
            p.a0 = p.b0 = p.e = l.s[k];
            p.d = l.p[k];
        }));
        TRY(symmetric(stage + 2, k, [&](Product &p, const Layout &l) {
            p.a0 = l.p[k];
            p.b0 = l.s[k];
            p.d = l.t;
        }));
        TRY(symmetric(stage + 3, k, [&](Product &p, const Layout &l) {
            p.a0 = l.t;
            p.b0 = l.p[k];
            p.d = l.s[k];
        }));
        TRY(symmetric(stage + 4, k, [&](Product &p, const Layout &l) {
            p.a0 = p.b0 = l.s[k];
            if (!f_.q.square) p.e = l.s[k];
            p.d = l.t;
        }));
        TRY(symmetric(stage + 5, k, [&](Product &p, const Layout &l) {
            p.a0 = l.t;
            p.b0 = l.p[k];
            p.d = l.s[k];
        }));
        return advance(stage + 6, k, k + 2, from, from ^ 1, [&](const Layout &l) { return l.s[k]; });
    }

    // Everything between the products with X of two steps at once, in one launch.
    bool thin() const {
        return std::all_of(b_.shapes.begin(), b_.shapes.end(),
                           [](const Batch::Shape &s) { return s.s <= kThin; });
    }

    int squares(int stage, int k) {
        SquareArgs a{};
        a.ws = c_.ws;
        a.factors = (const Factor *)(c_.ws + head_.factors);
        a.stages = stages_;
        a.stage = stage;
        const int64_t grid = shapes(a.sh, [&](const Batch::Shape &s, int g) {
            a.off[g] = s.lay.s[k];
            return (int64_t)1;
        });
        return launch(square_kernel, grid, 256, c_.stream, a);
    }

    int backwardStep(int k) {
        const int from = (steps_ - 1 - k) & 1, stage = kStepFactors * steps_ + 3 * k;
        TRY(product(stage, k, true, true, kToOperand, [&](Product &p, const Layout &l, int, int ld_w) {
            p.a0 = p.b1 = l.y[from];
            p.b0 = p.a1 = l.x[k];
            p.lda = p.ldb = ld_w;
            p.steps1 = 1;
            p.d = p.dt = l.m;
        }));
        TRY(product(stage + 1, k, true, true, kToOperand, [&](Product &p, const Layout &l, int ld_s, int) {
            p.a0 = p.b1 = l.m;
            if (!f_.q.square) p.e = l.m;
            p.b0 = p.a1 = l.s[k];
            p.lda = p.ldb = ld_s;
            p.steps1 = 1;
            p.d = p.dt = l.n;
        }));
        return product(stage + 2, k, true, false, k ? kToOperand : kToFloat,
                       [&](Product &p, const Layout &l, int ld_s, int) {
                           p.a0 = l.p[k];
                           p.b0 = l.yt[from];
                           p.a1 = l.n;
                           p.b1 = l.xt[k];
                           p.lda = p.ldb = ld_s;
            p.steps1 = 1;
                           p.d = k ? l.y[from ^ 1] : l.yf;
                           if (k) p.dt = l.yt[from ^ 1];
                       });
    }

    // Bounds of the cotangents from that of X_k on by its norm.
    int measure(int k) {
        TRY(dots<true>(k));
        f_.measured = k;
        return launch(factors_kernel, (int64_t)b_.mats.size(), 256, c_.stream, f_);
    }

    // <Y_0, X_0>, or the squares of the cotangent of X_k.
    template <bool SQUARE> int dots(int k) {
        TailArgs a = tailArgs();
        a.parts = (double *)(c_.ws + (SQUARE ? head_.parts_y : head_.parts));
        const int64_t grid = shapes(a.sh, [&](const Batch::Shape &s, int g) {
            a.y[g] = s.lay.yf;
            a.x[g] = SQUARE ? s.lay.y[(steps_ - k) & 1] : s.lay.x[0];
            const int64_t parts = std::min<int64_t>(kMaxParts, ((int64_t)s.s * s.w + 2047) / 2048);
            const int64_t cells = (s.s + 31) / 32 * (padded(s.w) / 32);
            a.per[g] = (cells + parts - 1) / parts;
            a.nparts[g] = (int)((cells + a.per[g] - 1) / a.per[g]);
            f_.nparts[g] = a.nparts[g];
            return (int64_t)a.nparts[g];
        });
        TRY(launch(dot_kernel<SQUARE>, grid, 256, c_.stream, a));
        return SQUARE ? 0 : tail(a);
    }

    TailArgs tailArgs() const {
        TailArgs a{};
        a.recs = recs();
        a.norms = (const MatNorm *)(c_.ws + head_.norms);
        a.ws = c_.ws;
        a.kept = c_.kept;
        return a;
    }

    int tail(TailArgs &a) {
        const int64_t grid = shapes(a.sh, [&](const Batch::Shape &s, int) {
            return padded(s.s) / 64 * (padded(s.w) / 64);
        });
        return withType(c_.dtype, [&](auto t) {
            using T = decltype(t);
            return launch(tail_kernel<T>, grid, 256, c_.stream, a);
        });
    }

    const Call &c_;
    const Batch &b_;
    const int steps_;
    const bool back_, keep_, few_;
    const int stages_;
    const Head head_;
    FactorArgs f_;
};

int run(const Call &call, size_t num, size_t workspace_bytes, size_t kept_bytes = 0) {
    if (call.dtype != TOA_F32 && call.dtype != TOA_F16 && call.dtype != TOA_BF16) return TOA_EDTYPE;
    Series series{};
    TRY(boundsOf(call.series, series));
    if (num == 0) return 0;
    if (!call.rows || !call.cols) return TOA_ENULL;
    std::vector<Batch> batches;
    std::vector<SmallBatch> smalls;
    int64_t bytes, kept;
    const Purpose purpose = call.what == kBackward ? (call.kept ? kGradientKept : kGradient)
                                                   : (call.kept ? kForwardKeep : kForward);
    TRY(plan(num, call.rows, call.cols, series, purpose, batches, smalls, bytes, kept));
    if (batches.empty() && smalls.empty()) return 0;
    if (!call.g || !call.out || (call.what != kOrthogonalize && !call.aux)) return TOA_ENULL;
    for (size_t i = 0; i < num; ++i)
        if (call.rows[i] && call.cols[i] &&
            (!call.g[i].data || !call.out[i].data || (call.aux && !call.aux[i].data) ||
             (call.momentum_dtype == TOA_I8 && (!call.scales || !call.scales[i]))))
            return TOA_ENULL;
    if (bytes && !call.ws) return TOA_ENULL;
    if (workspace_bytes < (size_t)bytes || ((uintptr_t)call.ws & 255)) return TOA_EWORKSPACE;
    if (call.kept && (kept_bytes < (size_t)kept || ((uintptr_t)call.kept & 255))) return TOA_EWORKSPACE;
    // (every launch of every batch is checked against the grid's limits before the first goes out)
    for (const Batch &b : batches)
        for (const auto &s : b.shapes)
            if (padded(s.s) / 64 * (padded(s.w) / 64) * (int64_t)b.mats.size() >
                std::numeric_limits<int>::max())
                return TOA_ESIZE;
    for (const SmallBatch &b : smalls) TRY(runSmall(call, b, series));
    for (const Batch &b : batches) TRY(Run(call, b, series).go());
    return 0;
}

// Nothing thrown in here may cross the C boundary.
template <typename F> int guarded(F fn) {
    try {
        return fn();
    } catch (...) {
        return (int)hipErrorOutOfMemory;
    }
}

// Of the workspace, or (`kept`) of the kept iterates.
size_t bytesOf(int dtype, size_t num, const int64_t *rows, const int64_t *cols,
               const toa_muon_series *q, Purpose purpose, bool kept, int *status) {
    int64_t bytes[2] = {};
    const int rc = guarded([&]() -> int {
        if (dtype != TOA_F32 && dtype != TOA_F16 && dtype != TOA_BF16) return TOA_EDTYPE;
        TRY(checkSeries(q));
        Series series{};
        TRY(boundsOf(*q, series));
        if (num && (!rows || !cols)) return TOA_ENULL;
        std::vector<Batch> batches;
        std::vector<SmallBatch> smalls;
        return plan(num, rows, cols, series, purpose, batches, smalls, bytes[0], bytes[1]);
    });
    if (status) *status = rc;
    return rc ? 0 : (size_t)bytes[kept];
}

// Launches over lists of flat arrays, 64 to a launch.
template <typename F>
int blocks(size_t num, const void *const *in, void *const *out, const float *const *scales,
           const size_t *n, F kernel, hipStream_t stream) {
    if (num == 0) return 0;
    if (!n) return TOA_ENULL;
    for (size_t i = 0; i < num; ++i) {
        if (!n[i]) continue;
        if (!in || !out || !scales || !in[i] || !out[i] || !scales[i]) return TOA_ENULL;
        if ((n[i] + 2047) / 2048 > (size_t)std::numeric_limits<int>::max() / 2) return TOA_ESIZE;
    }
    BlocksArgs a{};
    int64_t tiles = 0;
    for (size_t i = 0; i <= num; ++i) {
        const int64_t more = i < num ? (int64_t)((n[i] + 2047) / 2048) : 0;
        if (a.n && (i == num || a.n == kListMax || tiles + more > std::numeric_limits<int>::max())) {
            TRY(launch(kernel, tiles, 256, stream, a));
            a.n = 0;
            tiles = 0;
        }
        if (!more) continue;
        a.in[a.n] = in[i];
        a.out[a.n] = out[i];
        a.scales[a.n] = const_cast<float *>(scales[i]);
        a.count[a.n] = n[i];
        a.tile0[a.n] = (unsigned)tiles;
        tiles += more;
        ++a.n;
    }
    return 0;
}

}  // namespace

extern "C" {

int toa_muon_abi_version(void) { return 1; }

const char *toa_muon_error_string(int code) {
    switch (code) {
        case 0: return "success";
        case TOA_EDTYPE: return "toa_muon: unsupported dtype (float32, float16 and bfloat16 are served)";
        case TOA_ENULL: return "toa_muon: a required pointer is NULL";
        case TOA_ESIZE: return "toa_muon: a matrix is too large (a side beyond 2^20, or too many tiles)";
        case TOA_EVALUE: return "toa_muon: a number is out of range (steps, coefficients, eps, or a "
                                "hyper-parameter)";
        case TOA_EWORKSPACE: return "toa_muon: workspace too small or not 256-byte aligned";
        default: return code > 0 ? hipGetErrorString((hipError_t)code) : "toa_muon: unknown error";
    }
}

size_t toa_muon_orthogonalize_workspace(int dtype, size_t num, const int64_t *rows,
                                        const int64_t *cols, const toa_muon_series *series, int keep,
                                        int *status) {
    return bytesOf(dtype, num, rows, cols, series, keep ? kForwardKeep : kForward, false, status);
}

size_t toa_muon_backward_workspace(int dtype, size_t num, const int64_t *rows, const int64_t *cols,
                                   const toa_muon_series *series, int kept, int *status) {
    return bytesOf(dtype, num, rows, cols, series, kept ? kGradientKept : kGradient, false, status);
}

size_t toa_muon_kept_bytes(int dtype, size_t num, const int64_t *rows, const int64_t *cols,
                           const toa_muon_series *series, int *status) {
    return bytesOf(dtype, num, rows, cols, series, kForwardKeep, true, status);
}

int toa_muon_orthogonalize_multi(int dtype, size_t num, const int64_t *rows, const int64_t *cols,
                                 const toa_muon_view *in, const toa_muon_view *out,
                                 const toa_muon_series *series, void *kept, size_t kept_bytes,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&]() -> int {
        TRY(checkSeries(series));
        const Call c{kOrthogonalize, dtype, dtype, rows, cols, in, nullptr, out, nullptr, nullptr,
                     *series, (char *)workspace, (char *)kept, (hipStream_t)stream};
        return run(c, num, workspace_bytes, kept_bytes);
    });
}

int toa_muon_orthogonalize_backward_multi(int dtype, size_t num, const int64_t *rows,
                                          const int64_t *cols, const toa_muon_view *in,
                                          const toa_muon_view *grad_out,
                                          const toa_muon_view *grad_in,
                                          const toa_muon_series *series, const void *kept,
                                          size_t kept_bytes, void *workspace,
                                          size_t workspace_bytes, void *stream) {
    return guarded([&]() -> int {
        TRY(checkSeries(series));
        const Call c{kBackward, dtype, dtype, rows, cols, in, grad_out, grad_in, nullptr, nullptr,
                     *series, (char *)workspace, (char *)const_cast<void *>(kept),
                     (hipStream_t)stream};
        return run(c, num, workspace_bytes, kept_bytes);
    });
}

int toa_muon_step_multi(int dtype, int momentum_dtype, size_t num, const int64_t *rows,
                        const int64_t *cols, const toa_muon_view *out, const toa_muon_view *grads,
                        const toa_muon_view *momentum, float *const *scales,
                        const toa_muon_hyper *hyper, const toa_muon_series *series,
                        void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&]() -> int {
        TRY(checkSeries(series));
        if (!hyper) return TOA_ENULL;
        if (momentum_dtype != dtype && momentum_dtype != TOA_F32 && momentum_dtype != TOA_I8)
            return TOA_EDTYPE;
        if (!(hyper->momentum >= 0.0 && hyper->momentum < 1.0) ||
            hyper->adjust < TOA_MUON_UNIT || hyper->adjust > TOA_MUON_RMS ||
            (hyper->apply && !(std::isfinite(hyper->lr) && std::isfinite(hyper->weight_decay))))
            return TOA_EVALUE;
        const Call c{kStep, dtype, momentum_dtype, rows, cols, grads, momentum, out, scales, hyper,
                     *series, (char *)workspace, nullptr, (hipStream_t)stream};
        return run(c, num, workspace_bytes);
    });
}

int toa_muon_quantize_multi(int dtype, size_t num, const void *const *in, const size_t *n,
                            int8_t *const *codes, float *const *scales, void *stream) {
    return guarded([&]() -> int {
        return withType(dtype, [&](auto t) {
            return blocks(num, in, (void *const *)codes, (const float *const *)scales, n,
                          quantize_kernel<decltype(t)>, (hipStream_t)stream);
        });
    });
}

int toa_muon_dequantize_multi(int dtype, size_t num, const int8_t *const *codes,
                              const float *const *scales, const size_t *n, void *const *out,
                              void *stream) {
    return guarded([&]() -> int {
        return withType(dtype, [&](auto t) {
            return blocks(num, (const void *const *)codes, out, scales, n,
                          dequantize_kernel<decltype(t)>, (hipStream_t)stream);
        });
    });
}

}  // extern "C"
