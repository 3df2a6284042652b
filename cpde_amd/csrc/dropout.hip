// Dropout from a counter-based generator: y = keep ? x / (1 - p) : 0 (+ residual).
#include <cmath>

#include "sequence.hpp"

namespace cpde {
namespace {

// The four words of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, 2011): ten rounds
// of two 32 x 32 -> 64 products, their halves crossed and combined with the keys.
__device__ inline u32x4 philox(uint64_t counter, uint64_t seed) {
    uint32_t c0 = uint32_t(counter), c1 = uint32_t(counter >> 32), c2 = 0, c3 = 0;
    uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = uint64_t(0xD2511F53u) * c0, b = uint64_t(0xCD9E8D57u) * c2;
        c0 = uint32_t(b >> 32) ^ c1 ^ k0;
        c2 = uint32_t(a >> 32) ^ c3 ^ k1;
        c1 = uint32_t(b);
        c3 = uint32_t(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}

struct DropoutArgs {
    const void *x, *residual;
    void* y;
    int64_t x_stride, residual_stride, y_stride;
    uint64_t rows, columns, seed, offset;
    uint32_t threshold;
    int none;  // every element is dropped (the threshold is 2^32)
    float up;
};

template <class T>
__device__ inline T drop(const DropoutArgs& a, uint32_t word, T x, const T* residual) {
    // (a select, not a product: a dropped infinity or NaN leaves nothing)
    float v = word >= a.threshold && !a.none ? float(x) * a.up : 0.f;
    if (residual) v += float(*residual);
    return T(v);
}

// 16 bytes a lane.  Elements are counted through the rows, so a vector of a row
// whose length is a whole number of vectors starts on a counter; one row (a
// contiguous matrix) may end inside a vector.  Index: wide enough for the vectors.
// Bound: HBM.  A counter costs twenty 32 x 32 -> 64 products, 40 for the eight
// elements of a 16-bit vector, which the loads of other waves hide: on the
// measured card a copy of 256 MiB in 16-bit values runs at 5.7 TB/s, and with the
// generator at 5.6.  Results pass by the caches (262,144 x 256 in bf16 with a
// residual, then its gradient: 119 us, 123 through them).
template <class T, bool Residual, class Index>
__global__ __launch_bounds__(256) void dropout_wide_k(DropoutArgs a, Index vectors, Index per_row) {
    constexpr int N = 16 / sizeof(T);
    const Index step = Index(gridDim.x) * 256;
    for (Index i = Index(blockIdx.x) * 256 + threadIdx.x; i < vectors; i += step) {
        const Index row = a.rows == 1 ? 0 : i / per_row, at = (i - row * per_row) * N;
        const T* x = static_cast<const T*>(a.x) + int64_t(row) * a.x_stride + at;
        const T* residual = Residual ? static_cast<const T*>(a.residual) + int64_t(row) * a.residual_stride + at : nullptr;
        T* y = static_cast<T*>(a.y) + int64_t(row) * a.y_stride + at;
        const uint64_t counter = a.offset + uint64_t(i) * (N / 4);
        if (uint64_t(at) + N <= a.columns) {
            const vec<T, N> in = *reinterpret_cast<const vec<T, N>*>(x);
            vec<T, N> add, out;
            if (Residual) add = *reinterpret_cast<const vec<T, N>*>(residual);
#pragma unroll
            for (int q = 0; q < N / 4; ++q) {
                const u32x4 word = philox(counter + q, a.seed);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const T r = Residual ? T(add[4 * q + j]) : T(0.f);
                    out[4 * q + j] = drop<T>(a, word[j], T(in[4 * q + j]), Residual ? &r : nullptr);
                }
            }
            __builtin_nontemporal_store(__builtin_bit_cast(u32x4, out), reinterpret_cast<u32x4*>(y));
        } else {
            for (int j = 0; uint64_t(at) + j < a.columns; ++j)
                y[j] = drop<T>(a, philox(counter + j / 4, a.seed)[j % 4], x[j], residual ? residual + j : nullptr);
        }
    }
}

// Any strides and addresses: a lane takes one counter's four elements, which may
// lie in several rows.
template <class T>
__global__ __launch_bounds__(256) void dropout_any_k(DropoutArgs a) {
    const uint64_t count = a.rows * a.columns, step = uint64_t(gridDim.x) * 256;
    for (uint64_t q = uint64_t(blockIdx.x) * 256 + threadIdx.x; 4 * q < count; q += step) {
        const u32x4 word = philox(a.offset + q, a.seed);
        uint64_t row, column;
        if (count <= 0xffffffffull) {  // (a 32-bit division is a quarter of a 64-bit one)
            row = uint32_t(4 * q) / uint32_t(a.columns);
            column = uint32_t(4 * q) - uint32_t(row) * uint32_t(a.columns);
        } else {
            row = 4 * q / a.columns;
            column = 4 * q - row * a.columns;
        }
        for (int j = 0; j < 4 && 4 * q + j < count; ++j) {
            const T* residual =
                a.residual ? static_cast<const T*>(a.residual) + int64_t(row) * a.residual_stride + column : nullptr;
            static_cast<T*>(a.y)[int64_t(row) * a.y_stride + column] =
                drop<T>(a, word[j], static_cast<const T*>(a.x)[int64_t(row) * a.x_stride + column], residual);
            if (++column == a.columns) {
                column = 0;
                ++row;
            }
        }
    }
}

// Blocks of 256 lanes: at most 64 per CU, beyond which lanes take several vectors.
unsigned blocks_for(const Device& d, uint64_t lanes) {
    return unsigned(std::min<uint64_t>((lanes + 255) / 256, uint64_t(d.compute_units) * 64));
}

template <class T, bool Residual>
void launch_wide(Device& d, const DropoutArgs& a) {
    constexpr int N = 16 / sizeof(T);
    const uint64_t per_row = (a.columns + N - 1) / N, vectors = a.rows * per_row;
    const unsigned blocks = blocks_for(d, vectors);
    // (a loop's last step may pass the count by a grid's worth of lanes)
    if (vectors + uint64_t(blocks) * 256 < 0xffffffffull / N)
        hipLaunchKernelGGL((dropout_wide_k<T, Residual, uint32_t>), blocks, 256, 0, d.stream, a, uint32_t(vectors),
                           uint32_t(per_row));
    else
        hipLaunchKernelGGL((dropout_wide_k<T, Residual, uint64_t>), blocks, 256, 0, d.stream, a, vectors, per_row);
}

}  // namespace
}  // namespace cpde

using namespace cpde;

extern "C" int cpde_dropout(cpde_device* dev, int dtype, int64_t rows, int64_t columns, const cpde_rows* x,
                            const cpde_rows* residual, const cpde_rows* y, double probability, uint64_t seed,
                            uint64_t offset) {
    return guarded([&] {
        require(dev && x && y, "null argument");
        check_dtype(dtype);
        require(rows >= 0 && columns >= 0 && (columns == 0 || rows <= (int64_t(1) << 48) / columns),
                "invalid matrix size");
        require(probability >= 0 && probability <= 1, "a probability lies in 0..1");
        if (rows == 0 || columns == 0) return;
        require(x->data && y->data && (!residual || residual->data), "null tensor");
        require(x->stride >= 0 && (!residual || residual->stride >= 0), "negative stride");
        require(rows == 1 || y->stride >= columns, "output rows overlap");
        DropoutArgs a{};
        a.x = x->data;
        a.residual = residual ? residual->data : nullptr;
        a.y = y->data;
        a.x_stride = x->stride;
        a.residual_stride = residual ? residual->stride : 0;
        a.y_stride = y->stride;
        a.rows = uint64_t(rows);
        a.columns = uint64_t(columns);
        if (x->stride == columns && y->stride == columns && (!residual || residual->stride == columns)) {
            a.columns *= a.rows;
            a.rows = 1;
        }
        a.seed = seed;
        a.offset = offset;
        const double threshold = std::nearbyint(probability * 4294967296.0);
        a.none = threshold >= 4294967296.0;
        a.threshold = a.none ? 0xffffffffu : uint32_t(threshold);
        a.up = a.none ? 0.f : float(4294967296.0 / (4294967296.0 - threshold));
        const size_t size = type_bytes(dtype);
        const auto fits = [&](const cpde_rows* r) {
            return !r || (wide(r->data, a.rows == 1 ? 0 : r->stride, size));
        };
        const bool vectors = fits(x) && fits(y) && fits(residual) && (a.rows == 1 || columns * int64_t(size) % 16 == 0);
        flush_reduce(*dev);
        TraceScope trace(*dev, kTraceDropout, double(rows) * double(columns) * double(size) * (residual ? 3 : 2));
        with_type(dtype, [&](auto element) {
            using T = decltype(element);
            if (!vectors)
                hipLaunchKernelGGL((dropout_any_k<T>), blocks_for(*dev, (uint64_t(rows) * columns + 3) / 4), 256, 0,
                                   dev->stream, a);
            else if (residual) launch_wide<T, true>(*dev, a);
            else launch_wide<T, false>(*dev, a);
        });
        HIP_CHECK(hipGetLastError());
    });
}
