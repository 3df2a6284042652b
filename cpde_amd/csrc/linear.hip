// A layer's product with its bias, activation and residual, and its gradient.
#include <cmath>
#include <cstdio>

#include "product.hpp"

namespace cpde {
namespace {

// ---- activations ------------------------------------------------------------------------
__device__ inline float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }
__device__ inline float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + exp_fast(-z)); }
// The normal distribution's integral up to z, (1 + erf(z / sqrt 2)) / 2.  For 16-bit tensors by
// exp(z^2 / 2) times the integral up to -|z|, which is t P(t) with t = 1 / (1 + 0.2634 |z|) and P
// of degree six, fitted here for the least relative error over |z| <= 13.5 (5.4e-7): off by at most
// 4e-7, and, with its exponential's rounding, by 1e-5 of its value as far out as that is normal,
// so that small values have all the digits of their type.  It takes a third of the instructions of
// erfcf.
template <class T>
__device__ inline float normal_integral(float z) {
    if (sizeof(T) == 4) return 0.5f * erfcf(z * -0.70710678118654752440f);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.26339728f, fabsf(z), 1.f));
    float q = fmaf(-0.069694854f, t, 0.20668863f);
    q = fmaf(q, t, -0.079968646f);
    q = fmaf(q, t, 0.15077229f);
    q = fmaf(q, t, 0.07958568f);
    q = fmaf(q, t, 0.107690774f);
    q = fmaf(q, t, 0.10492611f);
    q *= t * __builtin_amdgcn_exp2f(z * z * -0.72134752044448170368f);
    return z < 0 ? q : 1 - q;
}

// Calls body with an activation's number as a constant.
template <class F>
__device__ __attribute__((always_inline)) inline void with_activation(int kind, F body) {
    switch (kind) {
        case CPDE_SIGMOID: return body(std::integral_constant<int, CPDE_SIGMOID>{});
        case CPDE_RELU: return body(std::integral_constant<int, CPDE_RELU>{});
        case CPDE_SILU: return body(std::integral_constant<int, CPDE_SILU>{});
        case CPDE_GELU: return body(std::integral_constant<int, CPDE_GELU>{});
        default: return;
    }
}
template <class T, int Kind>
__device__ inline float activate(float z) {
    if (Kind == CPDE_SIGMOID) return sigmoid(z);
    if (Kind == CPDE_RELU) return z < 0 ? 0.f : z;  // (a NaN stays one)
    if (Kind == CPDE_SILU) return z * sigmoid(z);
    return z * normal_integral<T>(z);
}
// Its derivative.
template <class T, int Kind>
__device__ inline float slope(float z) {
    if (Kind == CPDE_RELU) return z > 0 ? 1.f : 0.f;
    if (Kind == CPDE_GELU) return normal_integral<T>(z) + z * 0.39894228040143267794f * exp_fast(-0.5f * z * z);
    const float s = sigmoid(z);
    return Kind == CPDE_SILU ? s * (1 + z * (1 - s)) : s * (1 - s);
}

// ---- rows of a product on their way out ----------------------------------------------------
// y = activation(c + bias) + residual, and c + bias itself.  (Of a weight gradient: c, or
// with residual = y, onto what is there.)
template <class T>
struct LinearEpilogue {
    static constexpr bool kSymmetric = false, kAny = true;
    T *y, *pre;
    const T *bias, *residual;
    int64_t y_stride, pre_stride, residual_stride;
    int activation;
    // What a lane's columns have in common for all of its rows.
    struct Columns {
        float bias[8];
    };
    __device__ Columns columns(int, int n, int count) const {
        Columns c{};
        if (bias) read8(c.bias, bias + n, count);
        return c;
    }
    __device__ void row(const Columns& c, int, int m, int n, int count, float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += c.bias[j];
        if (pre) write8(pre + m * pre_stride + n, v, count);
        with_activation(activation, [&](auto kind) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = activate<T, decltype(kind)::value>(v[j]);
        });
        if (residual) {
            float r[8];
            read8(r, residual + m * residual_stride + n, count);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += r[j];
        }
        write8(y + m * y_stride + n, v, count);
    }
};

// Rows copied to whole 16-byte chunks, zeros behind their columns.  Where `again` is not 0:
// row r goes to rows r * every and r * every + again, and zeros follow the last one up to `all_rows`.
struct CopyArgs {
    int64_t stride, rows, all_rows;
    int columns, pitch, every, again;
};
template <class T>
__device__ inline void copy_chunks(const T* x, T* to, const CopyArgs& c, int64_t first_chunk, int64_t step) {
    const int per_row = c.pitch / 8;
    const int64_t all = c.all_rows * per_row;
    for (int64_t at = first_chunk; at < all; at += step) {
        const int64_t row = at / per_row;
        const int first = int(at - row * per_row) * 8;
        float v[8] = {};
        if (row < c.rows) read8(v, x + row * c.stride + first, min(8, c.columns - first));
        T* at_row = to + row * c.every * c.pitch + first;
        write8(at_row, v, 8);
        if (c.again) write8(at_row + int64_t(c.again) * c.pitch, v, 8);
    }
}

// ---- dz = dy * slope(pre) and its sums over the rows -----------------------------------------
// A workgroup takes 64 columns, eight a lane, of a strip of rows, 32 rows at a time; sums
// of a strip go to `part` [strip][columns], which linear_bias_k adds up in order.  Workgroups
// behind the last strip write what a dz of two values meets twice: weights, then x.
struct SlopeArgs {
    const void *dy, *pre;
    void* dz;       // null: not wanted (no activation)
    int64_t low;    // of what dz's rounding leaves, behind dz (0: not wanted)
    float* part;    // null: not wanted (no bias)
    int64_t dy_stride, pre_stride, rows;
    int columns, dz_stride, strip, strips, activation;
    const void* from[2];
    void* to[2];
    CopyArgs copy[2];
};
template <class T>
__global__ __launch_bounds__(256) void linear_slope_k(SlopeArgs a) {
    __shared__ float sums[32][64 + 8];
    if (int(blockIdx.y) >= a.strips) {
        const int64_t at = (int64_t(blockIdx.y - a.strips) * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
        const int64_t step = int64_t(gridDim.y - a.strips) * gridDim.x * 256;
#pragma unroll
        for (int i = 0; i < 2; ++i) copy_chunks(static_cast<const T*>(a.from[i]), static_cast<T*>(a.to[i]), a.copy[i], at, step);
        return;
    }
    const int lane = threadIdx.x & 7, row_lane = threadIdx.x >> 3, n = blockIdx.x * 64 + lane * 8;
    const int count = min(8, a.columns - n);
    const int64_t first = int64_t(blockIdx.y) * a.strip, last = min(first + a.strip, a.rows);
    float sum[8] = {};
    if (count > 0)
        for (int64_t m = first + row_lane; m < last; m += 32) {
            float v[8], z[8];
            read8(v, static_cast<const T*>(a.dy) + m * a.dy_stride + n, count);
            if (a.dz) {
                read8(z, static_cast<const T*>(a.pre) + m * a.pre_stride + n, count);
                with_activation(a.activation, [&](auto kind) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] *= slope<T, decltype(kind)::value>(z[j]);
                });
                T* to = static_cast<T*>(a.dz) + m * a.dz_stride + n;
                write8(to, v, 8);  // (zeros behind the columns)
                if (a.low) {
                    float left[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float high = float(T(v[j]));
                        left[j] = isfinite(high) ? v[j] - high : 0.f;
                    }
                    write8(to + a.low, left, 8);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += v[j];
        }
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[row_lane][lane * 8 + j] = sum[j];
    __syncthreads();
    if (threadIdx.x < 64 && blockIdx.x * 64 + threadIdx.x < unsigned(a.columns)) {
        float total = 0;
        for (int r = 0; r < 32; ++r) total += sums[r][threadIdx.x];
        a.part[int64_t(blockIdx.y) * a.columns + blockIdx.x * 64 + threadIdx.x] = total;
    }
}
// The strips' sums in order: 16 columns and 64 runs of strips a workgroup.
template <class T>
__global__ __launch_bounds__(1024) void linear_bias_k(const float* part, int strips, int columns, T* dbias, int accumulate) {
    __shared__ float sums[64][17];
    const int in = threadIdx.x & 15, run = threadIdx.x >> 4, n = blockIdx.x * 16 + in;
    const int per = (strips + 63) / 64;
    float total = 0;
    if (n < columns)
        for (int s = run * per; s < min(strips, (run + 1) * per); ++s) total += part[int64_t(s) * columns + n];
    sums[run][in] = total;
    __syncthreads();
    if (run || n >= columns) return;
    for (int r = 1; r < 64; ++r) total += sums[r][in];
    dbias[n] = T(accumulate ? float(dbias[n]) + total : total);
}

// ---- plans ---------------------------------------------------------------------------------
struct Linear {
    Device* dev = nullptr;
    int dtype = 0, inputs = 0, outputs = 0, activation = 0, backward = 0;
    int64_t rows = 0;
    char* work = nullptr;
    size_t a_copy = 0, b_copy = 0, dz = 0, twice[2] = {}, part = 0, bias_part = 0;  // places in the workspace
};
constexpr int64_t kMostRows = int64_t(1) << 30;
constexpr int kMostWidth = 1 << 24;
constexpr int kStrips = 256;  // of a bias's gradient
// Gradients of at most kFew values, from matrices of at most kFewInner, take a 16-bit dz as a
// sum of two values (the inner axis twice as long, its other operand written twice by
// linear_slope_k), and are as exact as the type.  Such calls wait for launches more than for
// products (256 -> 256, 256 rows: 12.9 us for 10.9; 128 -> 128, 1,000 rows: 16.4 for 12.6; 64 -> 64,
// 16,384 rows: 32.5 for 27.3).  Beyond, dz is rounded once and the products run at
// the matrix units' rate: the results lie 1.4 times as far from the exact ones.
constexpr int64_t kFew = 1 << 17, kFewInner = 1 << 20;

int pitch_of(int64_t columns) { return int((columns + 7) / 8 * 8); }

template <class T>
__global__ __launch_bounds__(256) void linear_copy_k(const T* x, T* to, CopyArgs c) {
    copy_chunks(x, to, c, int64_t(blockIdx.x) * 256 + threadIdx.x, int64_t(gridDim.x) * 256);
}
template <class T>
void copy_rows(Device& d, const void* x, T* to, const CopyArgs& c) {
    const int64_t chunks = c.all_rows * (c.pitch / 8);
    const unsigned blocks = unsigned(std::max<int64_t>(1, std::min<int64_t>((chunks + 255) / 256, int64_t(d.compute_units) * 32)));
    hipLaunchKernelGGL((linear_copy_k<T>), blocks, 256, 0, d.stream, static_cast<const T*>(x), to, c);
    HIP_CHECK(hipGetLastError());
}

// C[m][n] of a plan's product: operands by their rows, which AK and BK say the order of.
struct Sides {
    const void *a, *b;
    int64_t a_stride, b_stride, m, k;
    int n;
    bool a_whole, b_whole;  // its rows go on in zeros to whole chunks
};
// A product of a plan's, as it is launched, and the operands that are copied for it before.
struct Prepared {
    Product product;
    struct {
        const void* from;  // (null: not copied)
        void* to;
        CopyArgs args;
    } copy[2];
};
template <bool AK, bool BK, class T>
Prepared prepare(const Linear& p, const Sides& s) {
    const Device& d = *p.dev;
    Prepared r{};
    ProductArgs args{};
    args.m = int(s.m);
    args.n = s.n;
    args.k = int(s.k);
    args.batch = 1;
    args.part = reinterpret_cast<float*>(p.work + p.part);
    args.a = product_operand(s.a, s.a_stride, s.a_whole ? s.a_stride : AK ? s.k : s.m, sizeof(T));
    args.b = product_operand(s.b, s.b_stride, s.b_whole ? s.b_stride : BK ? s.k : s.n, sizeof(T));
    // Operands that are not whole chunks come through registers, 64 x 64 tiles at a time, where the
    // product is small or few tiles share them; else they are copied to whole chunks first, for larger
    // tiles (a plan whose widths are not whole eights has room for it).  2,047 -> 2,047: 256 rows bf16
    // 13.8 us through registers, 19.2 copied, f32 31.6 and 35.9; 512 rows 20.0 and 25.1, 71.0 and 47.8;
    // 2,048 rows 47.8 and 40.9, 155 and 116.  130 rows, 2,047 -> 8,191: 27.5 and 31.5, 67 and 82.
    const int64_t m_tiles = ceil_div(s.m, 64), n_tiles = ceil_div(s.n, 64), deep = ceil_div(s.k, kDepth<T>);
    const bool shared = std::min(m_tiles, n_tiles) > 3 && deep * m_tiles * n_tiles > 56 * int64_t(d.compute_units);
    if ((!args.a.wide || !args.b.wide) && p.a_copy && shared) {
        const auto copy = [&](int i, Operand& o, const void* x, int64_t stride, int64_t rows, int64_t columns, size_t place) {
            if (o.wide) return;
            const int pitch = pitch_of(columns);
            r.copy[i] = {x, p.work + place, {stride, rows, rows, int(columns), pitch, 1, 0}};
            o = product_operand(r.copy[i].to, pitch, pitch, sizeof(T));
        };
        copy(0, args.a, s.a, s.a_stride, AK ? s.m : s.k, AK ? s.k : s.m, p.a_copy);
        copy(1, args.b, s.b, s.b_stride, BK ? s.n : s.k, BK ? s.k : s.n, p.b_copy);
    }
    r.product = cut_for<T, AK, BK>(d, args);
    return r;
}
template <bool AK, bool BK, class T>
void launch(const Linear& p, const Prepared& r, const LinearEpilogue<T>& e) {
    for (const auto& c : r.copy)
        if (c.from) copy_rows<T>(*p.dev, c.from, static_cast<T*>(c.to), c.args);
    launch_product<T, AK, BK>(*p.dev, r.product, e);
}

// A gradient's products (those that are wanted), cut before the first launch: a refused call
// writes nothing.
struct Gradient {
    bool two_x, two_w;  // dz goes as two values
    const void* dz;     // (the plan's own: whole chunks, zeros behind the columns)
    int64_t dz_stride;
    Prepared dx, dweight;
};
template <class T>
Gradient prepare_gradient(const Linear& p, int64_t rows, const cpde_rows* x, const cpde_rows* weight, const cpde_rows& dy, bool dx,
                          bool dweight) {
    const bool bent = p.activation != CPDE_NONE;
    // (rows and widths to whole chunks are what is written)
    const int in = pitch_of(p.inputs), o = pitch_of(p.outputs);
    const bool two = bent && sizeof(T) == 2 && rows * o <= kFewInner;
    Gradient g{};
    g.two_x = two && dx && rows * in <= kFew && int64_t(o) * in <= kFewInner;
    g.two_w = two && dweight && int64_t(o) * in <= kFew && rows * in <= kFewInner;
    g.dz = bent ? p.work + p.dz : dy.data;
    g.dz_stride = !bent ? dy.stride : g.two_x || g.two_w ? 2 * o : o;
    if (dx)
        g.dx = prepare<true, false, T>(
            p, g.two_x ? Sides{g.dz, p.work + p.twice[0], g.dz_stride, in, rows, 2 * o, p.inputs, true, true}
                       : Sides{g.dz, weight->data, g.dz_stride, weight->stride, rows, p.outputs, p.inputs, bent, false});
    if (dweight)
        g.dweight = prepare<false, false, T>(
            p, g.two_w ? Sides{g.dz, p.work + p.twice[1], o, in, p.outputs, 2 * rows, p.inputs, true, true}
                       : Sides{g.dz, x->data, g.dz_stride, x->stride, p.outputs, rows, p.inputs, bent, false});
    return g;
}

// What runs for a product.
std::string describe(const Prepared& r) {
    const auto& [args, cut, wide] = r.product;
    if (r.product.empty()) return "nothing";
    std::string s = std::string(cut.side == 32 ? "product_run_k " : cut.side == 256 ? "product_large_k " : "product_k ") +
                    std::to_string(cut.side) + " splits " + std::to_string(args.splits);
    if (!wide) s += " through registers";
    if (r.copy[0].from || r.copy[1].from) s += " copied";
    return s;
}

// A matrix argument of `rows` x `columns`; an output's rows do not overlap.
void check_rows(const cpde_rows* r, int64_t rows, int64_t columns, bool output) {
    require(r, "null argument");
    if (!rows || !columns) return;
    require(r->data, "null tensor");
    require(r->stride >= 0 && r->stride <= int64_t(1) << 40, "invalid stride");
    require(!output || rows == 1 || r->stride >= columns, "output rows overlap");
}

}  // namespace
}  // namespace cpde

struct cpde_linear_s : cpde::Linear {};
using namespace cpde;

extern "C" {

int cpde_linear_create(cpde_device* dev, int dtype, int64_t rows, int inputs, int outputs, int activation, int backward,
                       cpde_linear** out) {
    return guarded([&] {
        require(dev && out, "null argument");
        *out = nullptr;
        check_dtype(dtype);
        require(activation >= CPDE_NONE && activation <= CPDE_GELU, "unknown activation");
        require(rows >= 0 && inputs >= 0 && outputs >= 0, "negative size");
        require(rows <= kMostRows && inputs <= kMostWidth && outputs <= kMostWidth, "too large a product");
        require(!dev->capturing, "a capture is open on this device");
        OnDevice on(*dev);
        auto p = std::make_unique<cpde_linear_s>();
        p->dev = dev;
        p->dtype = dtype;
        p->rows = rows;
        p->inputs = inputs;
        p->outputs = outputs;
        p->activation = activation;
        p->backward = backward != 0;
        size_t at = 0;
        const auto place = [&](size_t bytes) {
            const size_t here = at;
            at += (bytes + 255) / 256 * 256;
            return here;
        };
        if (inputs % 8 || outputs % 8) {
            // x or dy, and W or x, in whole chunks (the first place is never 0)
            const size_t size = type_bytes(dtype), in = pitch_of(inputs), o = pitch_of(outputs);
            place(256);
            p->a_copy = place(size * rows * (backward ? std::max(in, o) : in));
            p->b_copy = place(size * std::max(size_t(outputs) * in, backward ? size_t(rows) * in : 0));
        }
        if (backward && activation != CPDE_NONE) {
            const int64_t in = pitch_of(inputs), o = pitch_of(outputs);
            const bool short_type = dtype != CPDE_F32;  // (dz as two values, and what they meet written twice)
            p->dz = place(type_bytes(dtype) * (short_type ? std::max(rows * o, std::min(2 * rows * o, 2 * kFewInner)) : rows * o));
            if (short_type)
                for (int i = 0; i < 2; ++i) p->twice[i] = place(type_bytes(dtype) * std::min(2 * (i ? rows : o) * in, 2 * kFewInner));
        }
        if (backward) p->bias_part = place(sizeof(float) * kStrips * outputs);
        size_t part = product_part(dev->compute_units, 1, rows, outputs);
        if (backward)
            part = std::max({part, product_part(dev->compute_units, 1, rows, inputs),
                             product_part(dev->compute_units, 1, outputs, inputs)});
        p->part = place(sizeof(float) * part);
        HIP_CHECK(hipMalloc(&p->work, std::max<size_t>(at, 256)));
        *out = p.release();
    });
}

int cpde_linear_destroy(cpde_linear* linear) {
    return guarded([&] {
        if (!linear) return;
        OnDevice on(*linear->dev);
        sync_stream(*linear->dev, __LINE__);
        ++linear->dev->layout;
        HIP_CHECK(hipFree(linear->work));
        delete linear;
    });
}

int cpde_linear_info(cpde_linear* linear, int64_t rows, int aligned, char* text, size_t capacity) {
    return guarded([&] {
        require(linear && text && capacity, "null argument");
        const Linear& p = *linear;
        require(rows >= 0 && rows <= p.rows, "more rows than the plan's");
        with_type(p.dtype, [&](auto element) {
            using T = decltype(element);
            // (addresses are looked at, and not used)
            const auto of = [&](int columns) { return cpde_rows{reinterpret_cast<void*>(aligned ? 256 : 256 + sizeof(T)), columns}; };
            const cpde_rows x = of(p.inputs), dy = of(p.outputs);
            std::string s = "forward " + describe(prepare<true, true, T>(p, {x.data, x.data, x.stride, x.stride, rows, p.inputs, p.outputs, false, false}));
            if (p.backward) {
                const Gradient g = prepare_gradient<T>(p, rows, &x, &x, dy, true, true);
                s += ", dx " + describe(g.dx) + ", dweight " + describe(g.dweight);
            }
            std::snprintf(text, capacity, "%s", s.c_str());
        });
    });
}

int cpde_linear_forward(cpde_linear* linear, int64_t rows, const cpde_rows* x, const cpde_rows* weight, const void* bias,
                        const cpde_rows* residual, const cpde_rows* y, const cpde_rows* pre) {
    return guarded([&] {
        require(linear, "null argument");
        const Linear& p = *linear;
        require(rows >= 0 && rows <= p.rows, "more rows than the plan's");
        check_rows(x, rows, p.inputs, false);
        check_rows(weight, p.outputs, p.inputs, false);
        check_rows(y, rows, p.outputs, true);
        if (residual) check_rows(residual, rows, p.outputs, false);
        if (pre) check_rows(pre, rows, p.outputs, true);
        if (!rows || !p.outputs) return;
        Device& d = *p.dev;
        OnDevice on(d);
        flush_reduce(d);
        TraceScope trace(d, kTraceLinear, 2.0 * rows * p.inputs * p.outputs);
        with_type(p.dtype, [&](auto element) {
            using T = decltype(element);
            LinearEpilogue<T> e{};
            e.y = static_cast<T*>(y->data);
            e.y_stride = y->stride;
            e.bias = static_cast<const T*>(bias);
            if (residual) {
                e.residual = static_cast<const T*>(residual->data);
                e.residual_stride = residual->stride;
            }
            if (pre) {
                e.pre = static_cast<T*>(pre->data);
                e.pre_stride = pre->stride;
            }
            e.activation = p.activation;
            launch<true, true, T>(
                p, prepare<true, true, T>(p, {x->data, weight->data, x->stride, weight->stride, rows, p.inputs, p.outputs, false, false}), e);
        });
    });
}

int cpde_linear_backward(cpde_linear* linear, int64_t rows, const cpde_rows* x, const cpde_rows* weight,
                         const cpde_rows* pre, const cpde_rows* dy, const cpde_rows* dx, const cpde_rows* dweight,
                         void* dbias, int accumulate) {
    return guarded([&] {
        require(linear, "null argument");
        const Linear& p = *linear;
        require(p.backward, "the plan was created without a backward");
        require(rows >= 0 && rows <= p.rows, "more rows than the plan's");
        const bool bent = p.activation != CPDE_NONE;
        check_rows(dy, rows, p.outputs, false);
        if (bent) check_rows(pre, rows, p.outputs, false);
        if (dx) {
            check_rows(weight, p.outputs, p.inputs, false);
            check_rows(dx, rows, p.inputs, true);
        }
        if (dweight) {
            check_rows(x, rows, p.inputs, false);
            check_rows(dweight, p.outputs, p.inputs, true);
        }
        if (!dx && !dweight && !dbias) return;
        Device& d = *p.dev;
        OnDevice on(d);
        flush_reduce(d);
        TraceScope trace(d, kTraceLinearGradient, 2.0 * ((dx != nullptr) + (dweight != nullptr)) * rows * p.inputs * p.outputs);
        with_type(p.dtype, [&](auto element) {
            using T = decltype(element);
            const Gradient g = prepare_gradient<T>(p, rows, x, weight, *dy, dx != nullptr, dweight != nullptr);
            const int in = pitch_of(p.inputs), o = pitch_of(p.outputs);
            if ((bent || dbias) && p.outputs) {
                SlopeArgs a{};
                a.dy = dy->data;
                a.dy_stride = dy->stride;
                a.rows = rows;
                a.columns = p.outputs;
                a.activation = p.activation;
                if (bent) {
                    a.pre = pre->data;
                    a.pre_stride = pre->stride;
                    a.dz = p.work + p.dz;
                    a.dz_stride = int(g.dz_stride);
                    a.low = g.two_x || g.two_w ? o : 0;
                }
                if (dbias) a.part = reinterpret_cast<float*>(p.work + p.bias_part);
                // strips of 32 rows at least, and workgroups for the whole device
                const int column_blocks = ceil_div(p.outputs, 64);
                const int most = std::max(1, std::min<int>(kStrips, ceil_div(8 * d.compute_units, column_blocks)));
                a.strip = std::max(32, ceil_div(rows, most));
                const int strips = a.strips = std::max(1, ceil_div(rows, a.strip));
                // weights again below themselves, where dz and what it leaves stand side by side; rows of
                // x in turn with themselves, where those are rows of o
                if (g.two_x) {
                    a.from[0] = weight->data;
                    a.to[0] = p.work + p.twice[0];
                    a.copy[0] = {weight->stride, p.outputs, o, p.inputs, in, 1, o};
                }
                if (g.two_w) {
                    a.from[1] = x->data;
                    a.to[1] = p.work + p.twice[1];
                    a.copy[1] = {x->stride, rows, rows, p.inputs, in, 2, 1};
                }
                const int64_t chunks = std::max(g.two_x ? int64_t(o) * in : 0, g.two_w ? rows * in : 0) / 8;
                const int copiers = int(std::min<int64_t>(ceil_div(chunks, 256 * column_blocks), most));
                hipLaunchKernelGGL((linear_slope_k<T>), dim3(column_blocks, strips + copiers), 256, 0, d.stream, a);
                HIP_CHECK(hipGetLastError());
                if (dbias) {
                    hipLaunchKernelGGL((linear_bias_k<T>), ceil_div(p.outputs, 16), 1024, 0, d.stream, a.part, strips, p.outputs,
                                       static_cast<T*>(dbias), accumulate);
                    HIP_CHECK(hipGetLastError());
                }
            }
            if (dx) {
                LinearEpilogue<T> e{};
                e.y = static_cast<T*>(dx->data);
                e.y_stride = dx->stride;
                launch<true, false, T>(p, g.dx, e);
            }
            if (dweight) {
                LinearEpilogue<T> e{};
                e.y = static_cast<T*>(dweight->data);
                e.y_stride = dweight->stride;
                if (accumulate) {
                    e.residual = e.y;
                    e.residual_stride = e.y_stride;
                }
                launch<false, false, T>(p, g.dweight, e);
            }
        });
    });
}

}  // extern "C"
