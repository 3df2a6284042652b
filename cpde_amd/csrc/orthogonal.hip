// Matrices brought near the orthogonal ones of their singular vectors, and the step of an
// optimizer along them.
#include <cmath>

#include "product.hpp"

namespace cpde {
namespace {

// X <- a X + (b A + c A^2) X with A = X X^T (or X on the left of X^T X, whichever is
// smaller) takes every singular value s to a s + b s^3 + c s^5: from 0..1 into 0.68..1.13
// after a few steps, where s was not too small.
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
// The products' operands are f16, times 2^12: entries of X, A and b A + c A^2 lie below 4,
// and those down to 2^-26 stay in the type's normal range.  f32 and f16 matrices go as sums
// of two f16 values (22 bits; three of the four products, to 2^-22), so that the products
// stay as exact as the type; bf16 ones as one.  X itself is kept in floats: its
// roundings would pass through all later steps, which multiply small singular values by
// up to 485.
constexpr float kUp = 4096.f, kDown = 1.f / (4096.f * 4096.f);

struct Orthogonal {
    Device* dev = nullptr;
    int dtype = 0, count = 0, rows = 0, columns = 0, steps = 0;
    int blocks = 0;  // of a matrix's sums
    bool tall() const { return rows > columns; }
    int side() const { return std::min(rows, columns); }
    int planes() const { return dtype == CPDE_BF16 ? 1 : 2; }
    char* work = nullptr;
    size_t sums = 0, x = 0, x_half[2] = {}, gram = 0, gram_half = 0, poly = 0, part = 0;  // places in the workspace
};
int pitch_of(int columns) { return (columns + 7) / 8 * 8; }

template <class T>
struct Matrices {
    T* data;
    int64_t matrix, row;
    __device__ T* at(int m, int64_t r) const { return data + m * matrix + r * row; }
};

// What is brought near an orthogonal matrix: x, or the step that gradient and momentum
// give, which the first pass moves on.
template <class T>
struct Source {
    Matrices<const T> x;
    Matrices<float> momentum;  // (data null: none)
    float factor;
    int nesterov, wide;
    template <bool Move>
    __device__ void read(float (&v)[8], int matrix, int row, int first, int count) const {
        read8(v, x.at(matrix, row) + first, count, wide);
        if (!momentum.data) return;
        float m[8];
        float* at = momentum.at(matrix, row) + first;
        read8(m, at, count, wide);
        if (Move) {
#pragma unroll
            for (int j = 0; j < 8; ++j) m[j] = fmaf(factor, m[j], v[j]);
            write8(at, m, count, wide);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = nesterov ? fmaf(factor, m[j], v[j]) : m[j];
    }
};
struct Shape {
    int rows, columns, pitch, blocks;
};

__device__ inline double sum_block(double x) {
    __shared__ double sums[4];
#pragma unroll
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
    __syncthreads();
    return (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// Sums of squares of a matrix, a workgroup's each (and the momentum's move).
template <class T>
__global__ __launch_bounds__(256) void orthogonal_sums_k(Source<T> s, Shape p, double* sums) {
    const int per_row = p.pitch / 8;
    const int64_t all = int64_t(p.rows) * per_row;
    double total = 0;
    for (int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x; at < all; at += int64_t(p.blocks) * 256) {
        const int row = int(at / per_row), first = int(at - int64_t(row) * per_row) * 8;
        float v[8];
        s.template read<true>(v, blockIdx.y, row, first, min(8, p.columns - first));
        for (int j = 0; j < 8; ++j)
            if (first + j < p.columns) total += double(v[j]) * double(v[j]);
    }
    total = sum_block(total);
    if (threadIdx.x == 0) sums[blockIdx.y * p.blocks + blockIdx.x] = total;
}

// Eight values as f16, or as the sums of two, times 2^12.
template <int PLANES>
__device__ inline void write_halves(_Float16* to, int64_t plane, const float (&v)[8]) {
    vec<_Float16, 8> hi, lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float up = v[j] * kUp;
        hi[j] = _Float16(up);
        lo[j] = _Float16(up - float(hi[j]));
    }
    *reinterpret_cast<vec<_Float16, 8>*>(to) = hi;
    if (PLANES == 2) *reinterpret_cast<vec<_Float16, 8>*>(to + plane) = lo;
}

// X = x / |x|, in floats and as the products' operand; columns past the last are zeros.
template <class T, int PLANES>
__global__ __launch_bounds__(256) void orthogonal_scale_k(Source<T> s, Shape p, const double* sums, float* x, _Float16* half,
                                                          int64_t plane) {
    double total = 0;
    for (int i = threadIdx.x; i < p.blocks; i += 256) total += sums[blockIdx.y * p.blocks + i];
    total = sum_block(total);
    const double down = total > 0 ? 1 / sqrt(total) : total;  // (a NaN stays one)
    const int per_row = p.pitch / 8;
    const int64_t all = int64_t(p.rows) * per_row;
    for (int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x; at < all; at += int64_t(gridDim.x) * 256) {
        const int row = int(at / per_row), first = int(at - int64_t(row) * per_row) * 8;
        float v[8];
        s.template read<false>(v, blockIdx.y, row, first, min(8, p.columns - first));
        for (int j = 0; j < 8; ++j) v[j] = first + j < p.columns ? float(v[j] * down) : 0.f;
        const int64_t to = (int64_t(blockIdx.y) * p.rows + row) * p.pitch + first;
        write8(x + to, v, 8, true);
        write_halves<PLANES>(half + to, plane, v);
    }
}

// A from its product.  With one plane an operand, what is squared is A - 1: near the end A
// is, and the rounding of what differs from it is the smaller by as much.
template <int PLANES>
struct GramEpilogue {
    float* gram;
    _Float16* half;
    int64_t plane;
    int side, pitch;
    __device__ void row(int batch, int m, int n, int count, float (&v)[8]) const {
        const int64_t at = (int64_t(batch) * side + m) * pitch + n;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < count ? v[j] * kDown : 0.f;
        write8(gram + at, v, 8, true);
        if (PLANES == 1)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] -= m == n + j ? 1.f : 0.f;
        write_halves<PLANES>(half + at, plane, v);
    }
};
// b A + c A^2 from the square of A (or of A - 1, less 1 - 2 A).
template <int PLANES>
struct PolyEpilogue {
    const float* gram;
    _Float16* half;
    int64_t plane;
    int side, pitch;
    __device__ void row(int batch, int m, int n, int count, float (&v)[8]) const {
        const int64_t at = (int64_t(batch) * side + m) * pitch + n;
        float a[8];
        read8(a, gram + at, 8, true);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float square = v[j] * kDown;
            if (PLANES == 1) square += 2 * a[j] - (m == n + j ? 1.f : 0.f);
            v[j] = j < count ? kB * a[j] + kC * square : 0.f;
        }
        write_halves<PLANES>(half + at, plane, v);
    }
};
// The next X; after the last step out, or the weights' step along it.
template <class T, int PLANES>
struct StepEpilogue {
    float* x;
    _Float16* half;  // null: the last step
    int64_t plane;
    int rows, pitch, wide, update;
    Matrices<T> out;
    float keep, rate;  // weights <- keep weights - rate X
    __device__ void row(int batch, int m, int n, int count, float (&v)[8]) const {
        const int64_t at = (int64_t(batch) * rows + m) * pitch + n;
        float old[8];
        read8(old, x + at, 8, true);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < count ? kA * old[j] + v[j] * kDown : 0.f;
        if (half) {
            write8(x + at, v, 8, true);
            write_halves<PLANES>(half + at, plane, v);
            return;
        }
        T* to = out.at(batch, m) + n;
        if (update) {
            float w[8];
            read8(w, to, count, wide);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = keep * w[j] - rate * v[j];
        }
        write8(to, v, count, wide);
    }
};

// ---- on the host ----------------------------------------------------------------------------
const Planes kOne = {1, 0, 0};
const Planes kTwo = {3, 0b00'01'00, 0b00'00'01};  // (high and low, low and high, high and high)

void check_matrices(const Orthogonal& p, const cpde_matrices* x, bool output) {
    require(x, "null argument");
    if (!p.count || !p.rows || !p.columns) return;
    require(x->data, "null tensor");
    require(x->matrix >= 0 && x->row >= 0, "negative stride");
    require(x->matrix <= int64_t(1) << 40 && x->row <= int64_t(1) << 40, "invalid stride");
    if (!output) return;
    require(p.rows == 1 || x->row >= p.columns, "output elements overlap");
    require(p.count == 1 || x->matrix >= (p.rows - 1) * (p.rows > 1 ? x->row : 0) + p.columns, "output elements overlap");
}
template <class T>
Matrices<T> matrices(const cpde_matrices* x) {
    return {static_cast<T*>(x->data), x->matrix, x->row};
}
bool wide_matrices(const cpde_matrices* x, size_t size) {
    return wide(x->data, x->row, size) && wide(x->data, x->matrix, size);
}

template <class T, int PLANES>
void run(const Orthogonal& p, const Source<T>& source, StepEpilogue<T, PLANES> last) {
    Device& d = *p.dev;
    const int pitch = pitch_of(p.columns), side = p.side(), side_pitch = pitch_of(side);
    const int64_t plane = int64_t(p.count) * p.rows * pitch, side_plane = int64_t(p.count) * side * side_pitch;
    const auto at = [&](size_t place) { return p.work + place; };
    double* sums = reinterpret_cast<double*>(at(p.sums));
    float *x = reinterpret_cast<float*>(at(p.x)), *gram = reinterpret_cast<float*>(at(p.gram));
    _Float16 *x_half[2] = {reinterpret_cast<_Float16*>(at(p.x_half[0])), reinterpret_cast<_Float16*>(at(p.x_half[1]))};
    _Float16 *gram_half = reinterpret_cast<_Float16*>(at(p.gram_half)), *poly = reinterpret_cast<_Float16*>(at(p.poly));
    const Shape shape{p.rows, p.columns, pitch, p.blocks};
    hipLaunchKernelGGL((orthogonal_sums_k<T>), dim3(p.blocks, p.count), 256, 0, d.stream, source, shape, sums);
    HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL((orthogonal_scale_k<T, PLANES>), dim3(p.blocks, p.count), 256, 0, d.stream, source, shape, sums, x,
                       x_half[0], plane);
    HIP_CHECK(hipGetLastError());
    const auto operand = [&](const _Float16* data, int rows, int columns, int64_t plane_) {
        Operand o = product_operand(data, columns, columns, 2);
        o.plane = 2 * plane_;
        o.batch = int64_t(2) * rows * columns;
        return o;
    };
    ProductArgs g{};
    g.batch = p.count;
    g.planes = PLANES == 2 ? kTwo : kOne;
    g.part = reinterpret_cast<float*>(at(p.part));
    for (int step = 0; step < p.steps; ++step) {
        const Operand xs = operand(x_half[step & 1], p.rows, pitch, plane);
        const Operand as = operand(gram_half, side, side_pitch, side_plane), ps = operand(poly, side, side_pitch, side_plane);
        ProductArgs q = g;
        q.m = q.n = side;
        q.a = q.b = xs;
        q.k = p.tall() ? p.rows : p.columns;
        const GramEpilogue<PLANES> ge{gram, gram_half, side_plane, side, side_pitch};
        if (p.tall()) launch_product<_Float16, false, false>(d, q, ge);
        else launch_product<_Float16, true, true>(d, q, ge);
        q.a = q.b = as;
        q.k = side;
        launch_product<_Float16, true, true>(d, q, PolyEpilogue<PLANES>{gram, poly, side_plane, side, side_pitch});
        q.m = p.rows;
        q.n = p.columns;
        StepEpilogue<T, PLANES> se = last;
        se.x = x;
        se.half = step + 1 < p.steps ? x_half[(step + 1) & 1] : nullptr;
        se.plane = plane;
        se.rows = p.rows;
        se.pitch = pitch;
        if (p.tall()) {
            q.a = xs;
            q.b = ps;
            launch_product<_Float16, true, true>(d, q, se);
        } else {
            q.a = ps;
            q.b = xs;
            launch_product<_Float16, true, false>(d, q, se);
        }
    }
}
template <class T>
void run_typed(const Orthogonal& p, const Source<T>& source, const cpde_matrices* out, bool update, float keep, float rate) {
    constexpr int kPlanes = std::is_same_v<T, bf16> ? 1 : 2;
    StepEpilogue<T, kPlanes> last{};
    last.out = matrices<T>(out);
    last.wide = wide_matrices(out, sizeof(T));
    last.update = update;
    last.keep = keep;
    last.rate = rate;
    run<T, kPlanes>(p, source, last);
}
// Operations of a call: three products a step, the symmetric two by halves.
double flops(const Orthogonal& p) {
    const double r = p.side(), c = std::max(p.rows, p.columns);
    return p.count * p.steps * (3 * r * r * c + r * r * r);
}

}  // namespace
}  // namespace cpde

struct cpde_orthogonal_s : cpde::Orthogonal {};
using namespace cpde;

extern "C" {

int cpde_orthogonal_create(cpde_device* dev, int dtype, int count, int rows, int columns, int steps, cpde_orthogonal** out) {
    return guarded([&] {
        require(dev && out, "null argument");
        *out = nullptr;
        check_dtype(dtype);
        require(count >= 0 && rows >= 0 && columns >= 0, "negative size");
        require(count <= 1024 && rows <= 1 << 20 && columns <= 1 << 20, "too many or too large matrices");
        require(steps >= 1 && steps <= 32, "1 to 32 steps");
        require(!dev->capturing, "a capture is open on this device");
        OnDevice on(*dev);
        auto p = std::make_unique<cpde_orthogonal_s>();
        p->dev = dev;
        p->dtype = dtype;
        p->count = count;
        p->rows = rows;
        p->columns = columns;
        p->steps = steps;
        const size_t pitch = pitch_of(columns), side = p->side(), side_pitch = pitch_of(p->side()), n = count;
        p->blocks = int(std::max<int64_t>(1, std::min<int64_t>(2048, int64_t(rows) * (pitch / 8) / 256)));
        size_t at = 0;
        const auto place = [&](size_t bytes) {
            const size_t here = at;
            at += (bytes + 255) / 256 * 256;
            return here;
        };
        p->sums = place(sizeof(double) * n * p->blocks);
        p->x = place(sizeof(float) * n * rows * pitch);
        for (auto& half : p->x_half) half = place(2 * p->planes() * n * rows * pitch);
        p->gram = place(sizeof(float) * n * side * side_pitch);
        p->gram_half = place(2 * p->planes() * n * side * side_pitch);
        p->poly = place(2 * p->planes() * n * side * side_pitch);
        p->part = place(sizeof(float) * std::max(product_part(dev->compute_units, count, side, side),
                                                 product_part(dev->compute_units, count, rows, columns)));
        HIP_CHECK(hipMalloc(&p->work, std::max<size_t>(at, 256)));
        *out = p.release();
    });
}

int cpde_orthogonal_destroy(cpde_orthogonal* orthogonal) {
    return guarded([&] {
        if (!orthogonal) return;
        OnDevice on(*orthogonal->dev);
        sync_stream(*orthogonal->dev, __LINE__);
        ++orthogonal->dev->layout;
        HIP_CHECK(hipFree(orthogonal->work));
        delete orthogonal;
    });
}

int cpde_orthogonal_forward(cpde_orthogonal* orthogonal, const cpde_matrices* x, const cpde_matrices* out) {
    return guarded([&] {
        require(orthogonal, "null argument");
        const Orthogonal& p = *orthogonal;
        check_matrices(p, x, false);
        check_matrices(p, out, true);
        if (!p.count || !p.rows || !p.columns) return;
        OnDevice on(*p.dev);
        flush_reduce(*p.dev);
        TraceScope trace(*p.dev, kTraceOrthogonal, flops(p));
        with_type(p.dtype, [&](auto element) {
            using T = decltype(element);
            Source<T> s{};
            s.x = matrices<const T>(x);
            s.wide = wide_matrices(x, sizeof(T));
            run_typed<T>(p, s, out, false, 0, 0);
        });
    });
}

int cpde_orthogonal_update(cpde_orthogonal* orthogonal, const cpde_matrices* gradient, const cpde_matrices* momentum,
                           const cpde_matrices* weight, float rate, float factor, float decay, int nesterov) {
    return guarded([&] {
        require(orthogonal, "null argument");
        const Orthogonal& p = *orthogonal;
        check_matrices(p, gradient, false);
        check_matrices(p, momentum, true);
        check_matrices(p, weight, true);
        require(std::isfinite(rate) && std::isfinite(factor) && std::isfinite(decay), "rate, factor and decay are finite");
        if (!p.count || !p.rows || !p.columns) return;
        OnDevice on(*p.dev);
        flush_reduce(*p.dev);
        TraceScope trace(*p.dev, kTraceOrthogonal, flops(p));
        with_type(p.dtype, [&](auto element) {
            using T = decltype(element);
            Source<T> s{};
            s.x = matrices<const T>(gradient);
            s.momentum = matrices<float>(momentum);
            s.factor = factor;
            s.nesterov = nesterov;
            s.wide = wide_matrices(gradient, sizeof(T)) && wide_matrices(momentum, sizeof(float));
            const double size = double(rate) * std::sqrt(std::max(1.0, double(p.rows) / p.columns));
            run_typed<T>(p, s, weight, true, float(1 - double(rate) * decay), float(size));
        });
    });
}

}  // extern "C"
