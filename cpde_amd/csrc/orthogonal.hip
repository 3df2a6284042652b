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
// and one value has its 11 bits down to 2^-26.  f32 and f16 matrices go as sums of two f16
// values, three of the four products: off by 2^-22 of an entry, or by 2^-37, the second one's
// smallest steps, where the entry is below 2^-15.  That is of matrices of norm one: the sums of
// (b A + c A^2) X take it `side` times, 2^-24 of X up to a side of 8,192, and X's own entries
// are 2^-13 or more in the mean up to 8,192 x 8,192.  So the products stay as exact as the type; bf16
// matrices go as one value.  X itself is kept as a sum of two whatever the
// type: its roundings pass through all later steps, which multiply small singular values by
// up to 485.  With one value an operand the diagonals D of A and of b A + c A^2 stay apart in
// 32 bits, and the operands hold zeros there: a row's diagonal is the largest of it, and
// alike in all rows of a matrix with even singular values, so that its rounding would move
// all of them one way (4 x 15 x 526: 0.0026 from the exact values for 0.0017, which is the
// type's own rounding).  Small matrices have them apart whatever the type (f32: half the error,
// for 0.8 us a step).  With A = D + O: A^2 = D^2 + D O + O D + O^2.
constexpr float kUp = 4096.f, kDown = 1.f / (4096.f * 4096.f);

// b A + c A^2 of an entry from A and A^2; with the diagonal apart from O^2.
template <bool Apart>
__device__ inline float poly_of(float a, float square, bool diagonal, float row, float column) {
    if (Apart) square += a * (diagonal ? a : row + column);
    return kB * a + kC * square;
}

struct Orthogonal {
    Device* dev = nullptr;
    int dtype = 0, count = 0, rows = 0, columns = 0, steps = 0;
    int blocks = 0;  // of a matrix's sums
    bool tall() const { return rows > columns; }
    int side() const { return std::min(rows, columns); }
    int planes() const { return dtype == CPDE_BF16 ? 1 : 2; }
    char* work = nullptr;
    // places in the workspace (diagonal: of A, then of b A + c A^2)
    size_t sums = 0, x[2] = {}, gram = 0, poly = 0, diagonal = 0, part = 0;
};
int pitch_of(int columns) { return (columns + 31) / 32 * 32; }  // (whole groups of pairs)

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
    int nesterov;
    template <bool Move>
    __device__ void read(float (&v)[8], int matrix, int row, int first, int count) const {
        read8(v, x.at(matrix, row) + first, count);
        if (!momentum.data) return;
        float m[8];
        float* at = momentum.at(matrix, row) + first;
        read8(m, at, count);
        if (Move) {
#pragma unroll
            for (int j = 0; j < 8; ++j) m[j] = fmaf(factor, m[j], v[j]);
            write8(at, m, count);
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

// Where eight values of a matrix of f16 (PLANES 1: and a second one, `plane` on, of what they
// leave) or of pairs stand, and how far on their second parts.
template <int PLANES>
__device__ inline int64_t half_at(int64_t row, int pitch, int n) {
    return PLANES == 1 ? row * pitch + n : 2 * row * pitch + (n / 32) * 64 + n % 32;
}
template <int PLANES>
__device__ inline int64_t second_of(int64_t plane) { return PLANES == 1 ? plane : 32; }
// Eight values as f16, times 2^12, and what they leave.
__device__ inline void write_halves(_Float16* to, int64_t second, bool both, const float (&v)[8]) {
    vec<_Float16, 8> hi, lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float up = v[j] * kUp;
        hi[j] = _Float16(up);
        lo[j] = _Float16(up - float(hi[j]));
    }
    *reinterpret_cast<vec<_Float16, 8>*>(to) = hi;
    if (both) *reinterpret_cast<vec<_Float16, 8>*>(to + second) = lo;
}
__device__ inline void read_halves(float (&v)[8], const _Float16* from, int64_t second, bool both) {
    const auto hi = *reinterpret_cast<const vec<_Float16, 8>*>(from);
    vec<_Float16, 8> lo = {};
    if (both) lo = *reinterpret_cast<const vec<_Float16, 8>*>(from + second);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float(hi[j]) + float(lo[j])) * (1.f / kUp);
}

// X = x / |x|; columns past the last are zeros.
template <class T, int PLANES>
__global__ __launch_bounds__(256) void orthogonal_scale_k(Source<T> s, Shape p, const double* sums, _Float16* x, int64_t plane) {
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
        write_halves(x + half_at<PLANES>(int64_t(blockIdx.y) * p.rows + row, p.pitch, first), second_of<PLANES>(plane), true, v);
    }
}

// What stands on the diagonal at a lane's eight columns.
struct Diagonal {
    float d[8];
};
// A from its product.
template <int PLANES>
struct GramEpilogue {
    static constexpr bool kSymmetric = true, kAny = false;
    _Float16* gram;
    float* diagonal;  // (of one plane)
    int side, pitch;
    __device__ int columns(int, int, int) const { return 0; }
    __device__ void row(int, int batch, int m, int n, int count, float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = j < count ? v[j] * kDown : 0.f;
            if (PLANES == 1 && m == n + j) {
                diagonal[batch * side + m] = v[j];
                v[j] = 0;
            }
        }
        write_halves(gram + half_at<PLANES>(int64_t(batch) * side + m, pitch, n), 32, PLANES == 2, v);
    }
};
// b A + c A^2 from the square of A (or of O).
template <int PLANES>
struct PolyEpilogue {
    static constexpr bool kSymmetric = true, kAny = false;
    const _Float16* gram;
    _Float16* poly;
    const float* diagonal;
    float* poly_diagonal;
    int side, pitch;
    __device__ Diagonal columns(int batch, int n, int count) const {
        Diagonal c = {};
        if (PLANES == 1 && count > 0) read8(c.d, diagonal + batch * side + n, count);
        return c;
    }
    __device__ void row(const Diagonal& column, int batch, int m, int n, int count, float (&v)[8]) const {
        const int64_t at = half_at<PLANES>(int64_t(batch) * side + m, pitch, n);
        float a[8];
        read_halves(a, gram + at, 32, PLANES == 2);
        const float row = PLANES == 1 ? diagonal[batch * side + m] : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool one = PLANES == 1 && m == n + j;
            v[j] = j < count ? poly_of<PLANES == 1>(one ? row : a[j], v[j] * kDown, one, row, column.d[j]) : 0.f;
            if (one) {
                poly_diagonal[batch * side + m] = v[j];
                v[j] = 0;
            }
        }
        write_halves(poly + at, 32, PLANES == 2, v);
    }
};
// The next X; after the last step out, or the weights' step along it.
template <class T, int PLANES>
struct StepEpilogue {
    static constexpr bool kSymmetric = false, kAny = false;
    const _Float16* x;
    _Float16* next;  // null: the last step
    const float* diagonal;  // of b A + c A^2, with one plane
    int64_t plane;
    int rows, side, pitch, update;
    bool tall;  // (A stands on the right)
    Matrices<T> out;
    float keep, rate;  // weights <- keep weights - rate X
    __device__ Diagonal columns(int batch, int n, int count) const {
        Diagonal c = {};
        if (PLANES == 1 && tall && count > 0) read8(c.d, diagonal + batch * side + n, count);
        return c;
    }
    __device__ void row(const Diagonal& column, int batch, int m, int n, int count, float (&v)[8]) const {
        const int64_t at = half_at<PLANES>(int64_t(batch) * rows + m, pitch, n), second = second_of<PLANES>(plane);
        float old[8];
        read_halves(old, x + at, second, true);
        const float row = PLANES == 1 && !tall ? diagonal[batch * side + m] : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < count ? (kA + (row + column.d[j])) * old[j] + v[j] * kDown : 0.f;
        if (next) {
            write_halves(next + at, second, true, v);
            return;
        }
        T* to = out.at(batch, m) + n;
        if (update) {
            float w[8];
            read8(w, to, count);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = keep * w[j] - rate * v[j];
        }
        write8(to, v, count);
    }
};

// ---- small matrices in one launch -----------------------------------------------------------
// A workgroup takes a matrix of at most 128 x 128, 64 x 256 or 32 x 512 (or higher than
// wide) through all steps: X and A (then b A + c A^2) stay in LDS as the products' operands,
// the matrix lying so that it is at least as wide as high; its sixteen waves hold a 32 x 32
// of X and of A in registers.  Symmetric products are made by the waves of the blocks on and
// below the diagonal and stored twice.  Bound: the products of one CU (128 x 128 f32: 1.3 us
// each at the matrix unit's rate) and the barriers between them: 8 us a step; in launches
// of their own the three products of a step take 13.
constexpr int kSmall = 128;
// X's row in LDS, in columns.
__host__ __device__ inline int small_width(int wide) { return wide <= 128 ? 128 : wide <= 256 ? 256 : 512; }
__host__ __device__ inline bool is_small(int rows, int columns) {
    const int high = rows < columns ? rows : columns, wide = rows < columns ? columns : rows;
    return wide <= 512 && high <= kSmall * kSmall / small_width(wide);
}
struct SmallArgs {
    int rows, columns, steps;  // as the caller has them
    int update;
    float keep, rate;
};
// Chunk `chunk` of row `row` of an f16 matrix in LDS whose rows are `pitch` bytes (whole
// 256s), turned so that both 16 rows' same chunk and four rows' 64 bytes lie in different banks.
__device__ inline int small_at(int pitch, int row, int chunk) {
    return row * pitch + ((chunk ^ (((row & 3) << 2) | ((row >> 2) & 3))) << 4);
}
__device__ inline Frag<_Float16> small_row(const char* matrix, int pitch, int block, int s, int lane) {
    return *reinterpret_cast<const Frag<_Float16>*>(matrix + small_at(pitch, 32 * block + (lane & 31), 2 * s + (lane >> 5)));
}
__device__ inline Frag<_Float16> small_column(const char* matrix, int pitch, int block, int s, int lane) {
    const int row = 16 * s + 8 * (lane >> 5) + ((lane & 15) >> 2), chunk = 4 * block + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4* at;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(matrix + small_at(pitch, row, chunk) + (lane & 1) * 8));
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(matrix + small_at(pitch, row + 4, chunk) + (lane & 1) * 8));
    return __builtin_bit_cast(Frag<_Float16>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <class T, int PLANES>
__global__ __launch_bounds__(1024) void orthogonal_small_k(Source<T> s, SmallArgs p, Matrices<T> out) {
    constexpr int kPlane = kSmall * 256, kThreads = 1024;  // bytes of a plane
    __shared__ __align__(16) char x_lds[2 * kPlane];       // X; at the end the result in floats
    __shared__ __align__(16) char g_lds[PLANES * kPlane];
    __shared__ double sums[16];
    __shared__ float diagonal[kSmall];  // of A, then of b A + c A^2
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5, matrix = blockIdx.x;
    const bool tall = p.rows > p.columns;
    const int high = min(p.rows, p.columns), wide = max(p.rows, p.columns);
    constexpr int kG = 2 * kSmall;                    // bytes of a row of A
    const int width = small_width(wide), kX = 2 * width;  // X's
    // the matrix, its size, and X in LDS (its transpose where it is tall), zeros around it
    for (int i = threadIdx.x; i < 2 * kPlane / 16; i += kThreads) *reinterpret_cast<u32x4*>(x_lds + i * 16) = u32x4{0, 0, 0, 0};
    const int per_row = (p.columns + 7) / 8, all = p.rows * per_row;
    constexpr int kMost = kSmall * kSmall / 8 / kThreads;
    float v[kMost][8];
    double total = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int at = i * kThreads + threadIdx.x, row = at / per_row, first = at % per_row * 8;
        const int count = at < all ? min(8, p.columns - first) : 0;
        for (int j = 0; j < 8; ++j) v[i][j] = 0;
        if (count > 0) s.template read<true>(v[i], matrix, row, first, count);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[i][j] = j < count ? v[i][j] : 0.f;
            total += double(v[i][j]) * double(v[i][j]);
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
    if (lane == 0) sums[wave] = total;
    __syncthreads();
    total = 0;
    for (int w = 0; w < 16; ++w) total += sums[w];
    const double down = total > 0 ? double(kUp) / sqrt(total) : total;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int at = i * kThreads + threadIdx.x, row = at / per_row, first = at % per_row * 8;
        if (at >= all) continue;
        vec<_Float16, 8> hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float up = float(v[i][j] * down);
            hi[j] = _Float16(up);
            lo[j] = _Float16(up - float(hi[j]));
        }
        if (!tall) {
            char* to = x_lds + small_at(kX, row, first / 8);
            *reinterpret_cast<vec<_Float16, 8>*>(to) = hi;
            *reinterpret_cast<vec<_Float16, 8>*>(to + kPlane) = lo;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (first + j >= high) continue;
                char* to = x_lds + small_at(kX, first + j, row / 8) + (row & 7) * 2;
                *reinterpret_cast<_Float16*>(to) = hi[j];
                *reinterpret_cast<_Float16*>(to + kPlane) = lo[j];
            }
        }
    }
    __syncthreads();
    // this wave's block of X, and of A: the first ten waves have one on or below the diagonal
    struct Block {
        int m, n, row, column;  // element e: this row, column + 8 (e / 4) + e % 4
    };
    const auto block = [&](int m, int n) { return Block{m, n, 32 * m + (lane & 31), 32 * n + 4 * half}; };
    int am, an;
    triangle_of(wave, am, an);
    const Block bx = block(wave / (width / 32), wave % (width / 32)), ba = block(am, an);
    const bool square = wave < 10 && 32 * am < high, live = 32 * bx.m < high && 32 * bx.n < wide;
    // a block as f16 into LDS; turned: its transpose as well
    const auto put = [&](char* to, int pitch, int planes, const Block& b, bool turned, const Acc& c) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            vec<_Float16, 4> hi, lo;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float up = c[4 * g + j] * kUp;
                hi[j] = _Float16(up);
                lo[j] = _Float16(up - float(hi[j]));
            }
            char* at = to + small_at(pitch, b.row, 4 * b.n + g) + 8 * half;
            *reinterpret_cast<vec<_Float16, 4>*>(at) = hi;
            if (planes == 2) *reinterpret_cast<vec<_Float16, 4>*>(at + kPlane) = lo;
            if (turned)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    char* other = to + small_at(pitch, b.column + 8 * g + j, b.row / 8) + (b.row & 7) * 2;
                    *reinterpret_cast<_Float16*>(other) = hi[j];
                    if (planes == 2) *reinterpret_cast<_Float16*>(other + kPlane) = lo[j];
                }
        }
    };
    // sum over k of A(m, k) B(n, k): rows of `a`, rows or columns of `b`
    const auto product = [&](const char* a, int a_pitch, const char* b, int b_pitch, const Block& at, int steps, auto rows) __attribute__((always_inline)) {
        Acc c = {};
        // (a step's fragments are read while the one before is multiplied; the last one reads its own again)
        Frag<_Float16> fb[2][PLANES], fa[2][PLANES];
        const auto read = [&](int k, int to) __attribute__((always_inline)) {
#pragma unroll
            for (int q = 0; q < PLANES; ++q) {
                fb[to][q] = decltype(rows)::value ? small_row(b + q * kPlane, b_pitch, at.n, k, lane)
                                                  : small_column(b + q * kPlane, b_pitch, at.n, k, lane);
                fa[to][q] = small_row(a + q * kPlane, a_pitch, at.m, k, lane);
            }
        };
        const auto multiply_step = [&](int from) __attribute__((always_inline)) {
            if (PLANES == 2) {
                c = multiply(fb[from][1 % PLANES], fa[from][0], c);
                c = multiply(fb[from][0], fa[from][1 % PLANES], c);
            }
            c = multiply(fb[from][0], fa[from][0], c);
        };
        read(0, 0);
        for (int k = 0; k < steps; k += 2) {
            read(min(k + 1, steps - 1), 1);
            multiply_step(0);
            read(min(k + 2, steps - 1), 0);
            if (k + 1 < steps) multiply_step(1);
        }
        return c;
    };
    Acc x, a, c;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const char* at = x_lds + small_at(kX, bx.row, 4 * bx.n + g) + 8 * half;
        const auto hi = *reinterpret_cast<const vec<_Float16, 4>*>(at), lo = *reinterpret_cast<const vec<_Float16, 4>*>(at + kPlane);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * g + j] = (float(hi[j]) + float(lo[j])) * (1.f / kUp);
    }
    const int side_steps = (high + 15) / 16, wide_steps = (wide + 15) / 16;
    const auto on_diagonal = [&](int e) { return ba.row == ba.column + 8 * (e >> 2) + (e & 3); };
    // a symmetric matrix's block into LDS; its diagonal apart, zeros in its place
    const auto put_square = [&](Acc v) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (on_diagonal(e)) {
                diagonal[ba.row] = v[e];
                v[e] = 0;
            }
        put(g_lds, kG, PLANES, ba, am != an, v);
    };
    for (int step = 0; step < p.steps; ++step) {
        if (square) {
            a = product(x_lds, kX, x_lds, kX, ba, wide_steps, std::true_type{});
            a *= kDown;
            put_square(a);
        }
        __syncthreads();
        if (square) {
            c = product(g_lds, kG, g_lds, kG, ba, side_steps, std::true_type{});
            const float row = diagonal[ba.row];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float column = diagonal[ba.column + 8 * (e >> 2) + (e & 3)];
                c[e] = poly_of<true>(a[e], c[e] * kDown, on_diagonal(e), row, column);
            }
        }
        __syncthreads();
        if (square) put_square(c);
        __syncthreads();
        if (live) {
            c = product(g_lds, kG, x_lds, kX, bx, side_steps, std::false_type{});
            x = (kA + diagonal[bx.row]) * x + kDown * c;
        }
        __syncthreads();
        if (step + 1 < p.steps) {
            if (live) put(x_lds, kX, 2, bx, false, x);
            __syncthreads();
        }
    }
    // out by whole rows, through LDS: 16-byte chunks turned with the row
    const auto float_at = [&](int row, int column) { return x_lds + row * 4 * width + (((column >> 2) ^ (row & 31)) << 4) + (column & 3) * 4; };
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const Quad four = {x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
        *reinterpret_cast<Quad*>(float_at(bx.row, bx.column + 8 * g)) = four;
    }
    __syncthreads();
    for (int at = threadIdx.x; at < all; at += kThreads) {
        const int row = at / per_row, first = at % per_row * 8, count = min(8, p.columns - first);
        float y[8], w[8] = {};
        if (!tall) {
            *reinterpret_cast<Quad*>(y) = *reinterpret_cast<const Quad*>(float_at(row, first));
            *reinterpret_cast<Quad*>(y + 4) = *reinterpret_cast<const Quad*>(float_at(row, first + 4));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = *reinterpret_cast<const float*>(float_at(first + j, row));
        }
        T* to = out.at(matrix, row) + first;
        if (p.update) {
            read8(w, to, count);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = p.keep * w[j] - p.rate * y[j];
        }
        write8(to, y, count);
    }
}

// ---- on the host ----------------------------------------------------------------------------
void check_matrices(const Orthogonal& p, const cpde_matrices* x, bool output) {
    require(x, "null argument");
    if (!p.count || !p.rows || !p.columns) return;
    require(x->data, "null tensor");
    require(x->matrix >= 0 && x->row >= 0, "negative stride");
    require(x->matrix <= int64_t(1) << 40 && x->row <= int64_t(1) << 40, "invalid stride");
    if (!output) return;
    // (either axis may be the inner one: matrices may take turns row by row)
    std::pair<int64_t, int64_t> axes[] = {{x->matrix, p.count}, {x->row, p.rows}};
    if (axes[0] > axes[1]) std::swap(axes[0], axes[1]);
    int64_t extent = p.columns;
    for (const auto& [stride, count] : axes) {
        if (count == 1) continue;
        require(stride >= extent, "output elements overlap");
        extent += stride * (count - 1);
    }
}
template <class T>
Matrices<T> matrices(const cpde_matrices* x) {
    return {static_cast<T*>(x->data), x->matrix, x->row};
}
template <class T, int PLANES>
void run(const Orthogonal& p, const Source<T>& source, StepEpilogue<T, PLANES> last) {
    Device& d = *p.dev;
    if (is_small(p.rows, p.columns)) {
        const SmallArgs a{p.rows, p.columns, p.steps, last.update, last.keep, last.rate};
        hipLaunchKernelGGL((orthogonal_small_k<T, PLANES>), unsigned(p.count), 1024, 0, d.stream, source, a, last.out);
        HIP_CHECK(hipGetLastError());
        return;
    }
    using Value = std::conditional_t<PLANES == 2, Pair, _Float16>;  // of the operands
    const int pitch = pitch_of(p.columns), side = p.side(), side_pitch = pitch_of(side);
    const auto at = [&](size_t place) { return reinterpret_cast<_Float16*>(p.work + place); };
    double* sums = reinterpret_cast<double*>(p.work + p.sums);
    float *diagonal = reinterpret_cast<float*>(p.work + p.diagonal), *poly_diagonal = diagonal + int64_t(p.count) * side;
    _Float16 *x[2] = {at(p.x[0]), at(p.x[1])}, *gram = at(p.gram), *poly = at(p.poly);
    const Shape shape{p.rows, p.columns, pitch, p.blocks};
    const int64_t plane = int64_t(p.count) * p.rows * pitch;
    hipLaunchKernelGGL((orthogonal_sums_k<T>), dim3(p.blocks, p.count), 256, 0, d.stream, source, shape, sums);
    HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL((orthogonal_scale_k<T, PLANES>), dim3(p.blocks, p.count), 256, 0, d.stream, source, shape, sums, x[0], plane);
    HIP_CHECK(hipGetLastError());
    const auto operand = [&](const _Float16* data, int rows, int columns) {
        Operand o = product_operand(data, columns, columns, sizeof(Value));
        o.batch = int64_t(sizeof(Value)) * rows * columns;
        return o;
    };
    // (an inner axis along rows goes to the end of their zeros)
    ProductArgs g{};
    g.batch = p.count;
    g.part = reinterpret_cast<float*>(p.work + p.part);
    for (int step = 0; step < p.steps; ++step) {
        const Operand xs = operand(x[step & 1], p.rows, pitch), as = operand(gram, side, side_pitch), ps = operand(poly, side, side_pitch);
        ProductArgs q = g;
        q.symmetric = 1;
        q.m = q.n = side;
        q.a = q.b = xs;
        q.k = p.tall() ? p.rows : pitch;
        const GramEpilogue<PLANES> ge{gram, diagonal, side, side_pitch};
        if (p.tall()) launch_product<Value, false, false>(d, q, ge);
        else launch_product<Value, true, true>(d, q, ge);
        q.a = q.b = as;
        q.k = side_pitch;
        launch_product<Value, true, true>(d, q, PolyEpilogue<PLANES>{gram, poly, diagonal, poly_diagonal, side, side_pitch});
        q.symmetric = 0;
        q.m = p.rows;
        q.n = p.columns;
        StepEpilogue<T, PLANES> se = last;
        se.x = x[step & 1];
        se.next = step + 1 < p.steps ? x[(step + 1) & 1] : nullptr;
        se.diagonal = poly_diagonal;
        se.side = side;
        se.tall = p.tall();
        se.plane = plane;
        se.rows = p.rows;
        se.pitch = pitch;
        if (p.tall()) {
            q.a = xs;
            q.b = ps;
            launch_product<Value, true, true>(d, q, se);
        } else {
            // (the last columns of b A + c A^2 meet rows of X that there are not: k ends with them)
            q.a = ps;
            q.b = xs;
            q.k = side;
            launch_product<Value, true, false>(d, q, se);
        }
    }
}
template <class T>
void run_typed(const Orthogonal& p, const Source<T>& source, const cpde_matrices* out, bool update, float keep, float rate) {
    constexpr int kPlanes = std::is_same_v<T, bf16> ? 1 : 2;
    StepEpilogue<T, kPlanes> last{};
    last.out = matrices<T>(out);
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
        // (rows of 2^20 pairs are the longest that products take: no call is refused once it has begun)
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
        if (!is_small(rows, columns)) {
            for (auto& x : p->x) x = place(2 * 2 * n * rows * pitch);
            p->gram = place(2 * p->planes() * n * side * side_pitch);
            p->poly = place(2 * p->planes() * n * side * side_pitch);
        }
        const size_t operands = at;
        if (operands) {
            p->sums = place(sizeof(double) * n * p->blocks);
            p->diagonal = place(sizeof(float) * 2 * n * side);
            p->part = place(sizeof(float) * std::max(product_part(dev->compute_units, count, side, side),
                                                 product_part(dev->compute_units, count, rows, columns)));
        }
        HIP_CHECK(hipMalloc(&p->work, std::max<size_t>(at, 256)));
        try {
            // (what stands behind the operands' columns is never written: zeros)
            if (operands) launch_fill(*dev, reinterpret_cast<float*>(p->work), operands / sizeof(float), 0.f);
        } catch (...) {
            (void)hipFree(p->work);
            throw;
        }
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
            const double size = double(rate) * std::sqrt(std::max(1.0, double(p.rows) / p.columns));
            run_typed<T>(p, s, weight, true, float(1 - double(rate) * decay), float(size));
        });
    });
}

}  // extern "C"
