// Matrix products on tiles: C[m][n] = sum over k of A(m, k) B(n, k), each operand with
// either of its axes contiguous, and an epilogue on rows of C before they are stored.
#pragma once
#include "sequence.hpp"

namespace cpde {
namespace {

// A matrix of a product: `stride` bytes from row to row.  Rows are m (or n) where k is
// contiguous, and k where m (or n) is.  A matrix may stand as several planes whose sum
// it is, `plane` bytes apart, and be one of a batch, `batch` bytes apart.  wide: its
// rows are read in whole 16-byte chunks, and its stride leaves a tile's offsets in 31 bits.
struct Operand {
    const char* data;
    int64_t stride, plane, batch;
    int wide;
};
// Products of planes that make up one of the matrices: A's and B's plane numbers, two bits
// a product from the lowest.
struct Planes {
    int count;
    uint32_t a, b;
};
struct ProductArgs {
    Operand a, b;
    int m, n, k, batch;
    int m_tiles, n_tiles;
    int splits, span;  // of the inner axis, and a split's tiles of it
    float* part;       // [split][batch][m][n] where there are several
    Planes planes;
};

typedef float Acc __attribute__((ext_vector_type(16)));
typedef float Quad __attribute__((ext_vector_type(4)));
template <class T>
using Frag = vec<T, 8>;

// A 32 x 32 tile: lane l holds column l % 32, rows 8 g + 4 (l / 32) + j in element
// 4 g + j.  A fragment: row (or column) l % 32, inner indices 8 (l / 32) + j.
__device__ inline Acc multiply(Frag<bf16> a, Frag<bf16> b, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline Acc multiply(Frag<_Float16> a, Frag<_Float16> b, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline Acc multiply(Frag<float> a, Frag<float> b, Acc c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// A value that is the same in every lane, where the compiler cannot see it.
__device__ inline int uniform(int i) { return __builtin_amdgcn_readfirstlane(i); }

// Tiles hold 128 bytes along k: 64 values of 16 bits, 32 floats.
constexpr int kTileBytes = 128;
template <class T>
constexpr int kDepth = kTileBytes / int(sizeof(T));

// A tile of `N` rows of an operand in LDS, in 16-byte chunks whose place in the row is
// turned with the row's number, so that the lanes that LDS serves in one cycle (16 of a
// 16-byte read: 64 banks) find their chunks in different banks:
// K (k contiguous): [N][kDepth]; two rows span the banks, so the place turns by row / 2
// (by row alone half of all cycles were conflicts);
// else: [kDepth][N]; a transposing read takes 64 bytes of four rows, which turn by 64 bytes.
template <class T, bool K, int N, int Threads>
struct TileSide {
    static constexpr int kChunk = 16 / int(sizeof(T)), kDeep = kDepth<T>;
    static constexpr int kRows = K ? N : kDeep, kChunks = (K ? kDeep : N) / kChunk;
    static constexpr int kRowBytes = kChunks * 16, kBytes = kRows * kRowBytes;
    static constexpr int kSlots = kRows * kChunks, kSteps = kSlots / Threads;
    static_assert(kSlots % Threads == 0, "whole steps");
    static constexpr uint32_t kNone = 0x80000000u;  // past every buffer: reads as zeros

    __device__ static int turn(int row) {
        if (K) return (row >> 1) & 7;
        if (sizeof(T) == 4) return (((row >> 3) & 1) << 3) & (kChunks - 1);
        return ((row & 3) << 2) & (kChunks - 1);
    }
    // Fragment of rows 32 block + lane % 32, inner indices 16 s + 8 (lane / 32) + j.
    __device__ static Frag<T> fragment(const char* tile, int block, int s, int lane) {
        const int half = lane >> 5;
        if constexpr (K && sizeof(T) == 2) {
            const int row = 32 * block + (lane & 31);
            return *reinterpret_cast<const Frag<T>*>(tile + row * kRowBytes + (((2 * s + half) ^ turn(row)) << 4));
        } else if constexpr (K) {
            const int row = 32 * block + (lane & 31);
            const char* p = tile + row * kRowBytes;
            const auto lo = *reinterpret_cast<const vec<T, 4>*>(p + (((4 * s + 2 * half) ^ turn(row)) << 4));
            const auto hi = *reinterpret_cast<const vec<T, 4>*>(p + (((4 * s + 2 * half + 1) ^ turn(row)) << 4));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        } else if constexpr (sizeof(T) == 2) {
            // Sixteen lanes read four k-rows of sixteen values (four lanes a row) and get
            // them back transposed, a column each.
            const int row = 16 * s + 8 * half + ((lane & 15) >> 2);
            const int chunk = 4 * block + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s4* at;
            // (four rows on, the turn is the same)
            const char* p = tile + row * kRowBytes + ((chunk ^ turn(row)) << 4) + (lane & 1) * 8;
            const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(p));
            const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(p + 4 * kRowBytes));
            return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int column = 32 * block + (lane & 31);
            Frag<T> f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = 16 * s + 8 * half + j;
                f[j] = *reinterpret_cast<const T*>(tile + row * kRowBytes + (((column >> 2) ^ turn(row)) << 4) + (column & 3) * 4);
            }
            return f;
        }
    }

    // ---- bringing tiles: rows first..first + N of the operand, inner indices from kDeep t
    uint32_t low, high;  // the address of the workgroup's first row (column), the same in every lane
    int64_t stride;
    int rows, k;         // rows (columns) from there on, inner indices in all

    __device__ void start(const Operand& o, int batch, int first, int all, int k_) {
        const uint64_t at = reinterpret_cast<uint64_t>(o.data) + batch * o.batch +
                            (K ? int64_t(first) * o.stride : int64_t(first) * int64_t(sizeof(T)));
        low = uniform(int(uint32_t(at)));
        high = uniform(int(uint32_t(at >> 32)));
        stride = o.stride;
        rows = all - first;
        k = k_;
    }
    __device__ uint64_t base(int64_t plane, int t) const {
        return ((uint64_t(high) << 32) | low) + plane + t * (K ? int64_t(kTileBytes) : kDeep * stride);
    }
    // Byte offset of a lane's chunk i of a tile with `left` inner indices.  Rows past the
    // last repeat it (their results are not stored); inner indices past the end are zeros.
    __device__ uint32_t place(int i, int left) const {
        const int slot = i * Threads + threadIdx.x, row = slot / kChunks, chunk = (slot % kChunks) ^ turn(row);
        if (K) return chunk * kChunk < left ? uint32_t(min(row, rows - 1)) * uint32_t(stride) + (chunk << 4) : kNone;
        return row < left ? uint32_t(row) * uint32_t(stride) + (min(chunk, (rows + kChunk - 1) / kChunk - 1) << 4) : kNone;
    }
    __device__ void places(uint32_t (&offset)[kSteps]) const {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) offset[i] = place(i, kDeep);
    }
    // From memory to LDS without registers, for operands of whole 16-byte chunks.  The
    // loads have arrived after loads_arrived() and a barrier.
    __device__ __attribute__((always_inline)) void load(char* tile, const uint32_t (&offset)[kSteps], int64_t plane, int t,
                                                        int wave) const {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's compiler does not know a buffer's type)
        const auto buffer = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base(plane, t)), 0, 0x7ffffff0, 0x00020000);
        const int left = k - t * kDeep;
        const auto bring = [&](int i, uint32_t at) __attribute__((always_inline)) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                buffer, (__attribute__((address_space(3))) void*)(tile + (i * Threads + wave * 64) * 16), 16, at, 0, 0, 0);
        };
        if (left >= kDeep) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) bring(i, offset[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) bring(i, place(i, left));
        }
#endif
    }
    // Value by value, for any other.
    __device__ void load_any(char* tile, int64_t plane, int t) const {
        const int left = k - t * kDeep;
        for (int i = 0; i < kSteps; ++i) {
            const int slot = i * Threads + threadIdx.x, row = slot / kChunks, first = ((slot % kChunks) ^ turn(row)) * kChunk;
            const T* p = reinterpret_cast<const T*>(base(plane, t) + int64_t(K ? min(row, rows - 1) : row) * stride);
            vec<T, kChunk> v;
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
                const bool there = K ? first + j < left : row < left && first + j < rows;
                v[j] = there ? p[first + j] : T(0.f);
            }
            *reinterpret_cast<vec<T, kChunk>*>(tile + slot * 16) = v;
        }
    }
};

__device__ inline void loads_arrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0), the other counters open

// Where a workgroup's tile lies.  Workgroups go to the 8 XCDs in turn, each with an L2 of
// its own: an XCD takes a run of neighbouring tiles, in bands of 8 tiles of m, so that
// those that run at once share rows of both operands.
__device__ inline void tile_of(int at, int count, int m_tiles, int n_tiles, int& tm, int& tn) {
    const int per = count / 8, over = count % 8, x = at % 8;
    at = x * per + min(x, over) + at / 8;
    const int band = at / (8 * n_tiles), height = min(8, m_tiles - 8 * band), in = at - band * 8 * n_tiles;
    tm = 8 * band + in % height;
    tn = in / height;
}

// Up to eight neighbouring values of a row, as floats.
template <class T>
__device__ inline void read8(float (&v)[8], const T* p, int count, bool wide) {
    constexpr int N = 16 / int(sizeof(T));
    if (wide && count == 8) {
#pragma unroll
        for (int part = 0; part < 8; part += N) {
            const auto in = *reinterpret_cast<const vec<T, N>*>(p + part);
#pragma unroll
            for (int j = 0; j < N; ++j) v[part + j] = float(in[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < count ? float(p[j]) : 0.f;
    }
}
template <class T>
__device__ inline void write8(T* p, const float (&v)[8], int count, bool wide) {
    constexpr int N = 16 / int(sizeof(T));
    if (wide && count == 8) {
#pragma unroll
        for (int part = 0; part < 8; part += N) {
            vec<T, N> out;
#pragma unroll
            for (int j = 0; j < N; ++j) out[j] = T(v[part + j]);
            *reinterpret_cast<vec<T, N>*>(p + part) = out;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) p[j] = T(v[j]);
    }
}

// What the kernels of products share: C's tile [BM][BN] by waves of [WM][WN] each, two
// tiles of either operand in LDS.
template <class T, bool AK, bool BK, int BM, int BN, int WM, int WN>
struct Tiles {
    static constexpr int kThreads = (BM / WM) * (BN / WN) * 64, kMB = WM / 32, kNB = WN / 32, kS = kDepth<T> / 16;
    using A = TileSide<T, AK, BM, kThreads>;
    using B = TileSide<T, BK, BN, kThreads>;
    static constexpr int kPitch = WN + 4, kStage = 32 * kPitch * 4;  // a wave's rows of C on their way out
    static constexpr int kTile = A::kBytes + B::kBytes, kOut = kThreads / 64 * kStage;
    static constexpr int kLds = 2 * kTile > kOut ? 2 * kTile : kOut;

    A a;
    B b;
    uint32_t a_offset[A::kSteps], b_offset[B::kSteps];
    int lane, wave, wm, wn, split, batch, m0, n0, t, t1, plane, steps;
    Acc acc[kMB][kNB];

    __device__ __attribute__((always_inline)) void start(const ProductArgs& p) {
        lane = threadIdx.x & 63;
        wave = uniform(threadIdx.x >> 6);
        wm = wave % (BM / WM);
        wn = wave / (BM / WM);
        split = blockIdx.y % p.splits;
        batch = blockIdx.y / p.splits;
        int tm, tn;
        tile_of(blockIdx.x, p.m_tiles * p.n_tiles, p.m_tiles, p.n_tiles, tm, tn);
        m0 = tm * BM;
        n0 = tn * BN;
        a.start(p.a, batch, m0, p.m, p.k);
        b.start(p.b, batch, n0, p.n, p.k);
        a.places(a_offset);
        b.places(b_offset);
        t = split * p.span;
        t1 = min((p.k + kDepth<T> - 1) / kDepth<T>, t + p.span);
        plane = 0;
        steps = max(0, t1 - t) * p.planes.count;
#pragma unroll
        for (int i = 0; i < kMB; ++i)
#pragma unroll
            for (int j = 0; j < kNB; ++j) acc[i][j] = Acc{};
    }
    // The next tile's loads.
    template <bool Any>
    __device__ __attribute__((always_inline)) void load(const ProductArgs& p, char* tile) {
        const int64_t pa = int64_t((p.planes.a >> (2 * plane)) & 3) * p.a.plane, pb = int64_t((p.planes.b >> (2 * plane)) & 3) * p.b.plane;
        if (Any && !p.a.wide) a.load_any(tile, pa, t);
        else a.load(tile, a_offset, pa, t, wave);
        if (Any && !p.b.wide) b.load_any(tile + A::kBytes, pb, t);
        else b.load(tile + A::kBytes, b_offset, pb, t, wave);
        if (++plane == p.planes.count) {
            plane = 0;
            ++t;
        }
    }
    __device__ __attribute__((always_inline)) void fragments(const char* tile, int s, Frag<T> (&fa)[kMB], Frag<T> (&fb)[kNB]) const {
#pragma unroll
        for (int i = 0; i < kMB; ++i) fa[i] = A::fragment(tile, wm * kMB + i, s, lane);
#pragma unroll
        for (int i = 0; i < kNB; ++i) fb[i] = B::fragment(tile + A::kBytes, wn * kNB + i, s, lane);
    }
    __device__ __attribute__((always_inline)) void products(const Frag<T> (&fa)[kMB], const Frag<T> (&fb)[kNB]) {
#pragma unroll
        for (int i = 0; i < kMB; ++i)
#pragma unroll
            for (int j = 0; j < kNB; ++j) acc[i][j] = multiply(fb[j], fa[i], acc[i][j]);
    }
    // Rows of C through LDS, so that eight neighbouring columns of a row are one lane's.
    template <class Epilogue>
    __device__ __attribute__((always_inline)) void finish(const ProductArgs& p, const Epilogue& e, char* lds) {
        float* stage = reinterpret_cast<float*>(lds + wave * kStage);
        constexpr int kLanes = WN / 8, kAtOnce = 64 / kLanes;
        const int half = lane >> 5;
#pragma unroll
        for (int i = 0; i < kMB; ++i) {
#pragma unroll
            for (int j = 0; j < kNB; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const Quad v = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                    *reinterpret_cast<Quad*>(stage + (lane & 31) * kPitch + 32 * j + 8 * g + 4 * half) = v;
                }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int r = 0; r < 32 / kAtOnce; ++r) {
                const int row = r * kAtOnce + lane / kLanes, column = (lane % kLanes) * 8;
                const int m = m0 + wm * WM + 32 * i + row, n = n0 + wn * WN + column;
                float v[8];
                *reinterpret_cast<Quad*>(v) = *reinterpret_cast<const Quad*>(stage + row * kPitch + column);
                *reinterpret_cast<Quad*>(v + 4) = *reinterpret_cast<const Quad*>(stage + row * kPitch + column + 4);
                if (m >= p.m || n >= p.n) continue;
                if (p.splits > 1)
                    write8(p.part + ((int64_t(split) * p.batch + batch) * p.m + m) * p.n + n, v, min(8, p.n - n), p.n % 4 == 0);
                else
                    e.row(batch, m, n, min(8, p.n - n), v);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
};

// The next tile's loads are under way while one is multiplied.  Any: operands of any
// alignment.
template <class T, bool AK, bool BK, int Side, int Wave, int PerSimd, bool Any, class Epilogue>
__global__ __launch_bounds__((Side / Wave) * (Side / Wave) * 64, PerSimd) void product_k(ProductArgs p, Epilogue e) {
    using C = Tiles<T, AK, BK, Side, Side, Wave, Wave>;
    __shared__ __align__(16) char lds[C::kLds];
    C c;
    c.start(p);
    // (the tiles read and written do not overlap, which the compiler has to know so as
    // not to wait for the loads under way before it reads)
    const auto step = [&](const char* __restrict__ tile) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < C::kS; ++s) {
            Frag<T> fa[C::kMB], fb[C::kNB];
            c.fragments(tile, s, fa, fb);
            c.products(fa, fb);
        }
    };
    if (c.steps) c.template load<Any>(p, lds);
    for (int i = 0; i < c.steps; ++i) {
        loads_arrived();
        __syncthreads();
        if (i + 1 < c.steps) c.template load<Any>(p, lds + ((i + 1) & 1) * C::kTile);
        step(lds + (i & 1) * C::kTile);
    }
    __syncthreads();
    c.finish(p, e, lds);
}

// Large products: 256 x 256 by eight waves, two on every SIMD, of which one multiplies while
// the other reads its fragments: the second four are half a tile's half behind the first,
// and barriers keep them there.
// A tile's buffer is written anew by loads issued when the first four have read the next
// one's first half and the second four, whose reads of it were waited for before the
// barrier in between, multiply.  Bound: matrix units, busy 64% of the cycles, at a clock
// that their power brings down from 2.4 to 2.0 GHz.
// Measured: 8192 x 8192 x 8192 bf16 857 us, 1,283 TFLOP/s; all waves in step 874 us (a large library
// product on the same card: 717 us).
template <class T, bool AK, bool BK, class Epilogue>
__global__ __launch_bounds__(512, 2) void product_large_k(ProductArgs p, Epilogue e) {
    using C = Tiles<T, AK, BK, 256, 256, 128, 64>;
    __shared__ __align__(16) char lds[C::kLds];
    C c;
    c.start(p);
    const bool second = c.wave >= 4;
    const auto barrier = [&]() __attribute__((always_inline)) {
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    if (c.steps) c.template load<false>(p, lds);
    loads_arrived();
    __syncthreads();
    if (second) barrier();
    for (int i = 0; i < c.steps; ++i) {
        const char* tile = lds + (i & 1) * C::kTile;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            Frag<T> fa[2][C::kMB], fb[2][C::kNB];
            c.fragments(tile, 2 * part, fa[0], fb[0]);
            c.fragments(tile, 2 * part + 1, fa[1], fb[1]);
            __builtin_amdgcn_sched_barrier(0);
            if (part == 0 && i + 1 < c.steps) c.template load<false>(p, lds + ((i + 1) & 1) * C::kTile);
            if (part == 1 && second) loads_arrived();
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the reads
            barrier();
            __builtin_amdgcn_s_setprio(1);
            c.products(fa[0], fb[0]);
            c.products(fa[1], fb[1]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            if (part == 1 && !second) loads_arrived();
            barrier();
        }
    }
    if (!second) barrier();
    __syncthreads();
    c.finish(p, e, lds);
}

// The splits of a product summed in order, eight columns a lane, and its epilogue.
template <class Epilogue>
__global__ __launch_bounds__(256) void product_join_k(ProductArgs p, Epilogue e) {
    const int per_row = (p.n + 7) / 8;
    const int64_t all = int64_t(p.batch) * p.m * per_row, at = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (at >= all) return;
    const int64_t row = at / per_row;  // of the batch's rows
    const int n = int(at - row * per_row) * 8, count = min(8, p.n - n), batch = int(row / p.m);
    float v[8] = {};
    for (int s = 0; s < p.splits; ++s) {
        float one[8];
        read8(one, p.part + (int64_t(s) * p.batch * p.m + row) * p.n + n, count, p.n % 4 == 0);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += one[j];
    }
    e.row(batch, int(row - int64_t(batch) * p.m), n, count, v);
}

// ---- on the host --------------------------------------------------------------------------
inline int ceil_div(int64_t a, int64_t b) { return int((a + b - 1) / b); }

// How a product is cut: the side of its tiles, and splits of its inner axis.
struct ProductCut {
    int side = 64, splits = 1, span = 1;
};
constexpr int kMostSplits = 64;
// depth: inner indices of all products of planes together.
inline ProductCut cut_product(int compute_units, int64_t batch, int64_t m, int64_t n, int64_t depth, int size, bool wide) {
    ProductCut c;
    const auto tiles = [&](int side) { return batch * ceil_div(m, side) * int64_t(ceil_div(n, side)); };
    if (wide && size == 2 && tiles(256) >= compute_units) c.side = 256;
    else if (wide && tiles(128) >= compute_units) c.side = 128;
    const int64_t have = std::max<int64_t>(1, tiles(c.side)), deep = (depth + kTileBytes / size - 1) / (kTileBytes / size);
    if (c.side < 256) c.splits = int(std::max<int64_t>(1, std::min<int64_t>({2 * compute_units / have, deep / 4, kMostSplits})));
    return c;
}
// Floats of ProductArgs::part that no call with up to `m` rows passes.
inline size_t product_part(int compute_units, int64_t batch, int64_t m, int64_t n) {
    return size_t(std::min<int64_t>(int64_t(2) * compute_units * 128 * 128, kMostSplits * batch * m * n));
}

// An operand of rows of `columns` values of `size` bytes.
inline Operand product_operand(const void* data, int64_t stride, int64_t columns, size_t size) {
    Operand o{};
    o.data = static_cast<const char*>(data);
    o.stride = stride * int64_t(size);
    o.wide = wide(data, stride, size) && columns * size % 16 == 0 && o.stride < (int64_t(1) << 22);
    return o;
}

// A launch of one of the kernels of tiles of `side`.
template <class K, class E>
void launch_tiles(Device& d, K kernel, int side, int threads, ProductArgs p, const E& e) {
    p.m_tiles = ceil_div(p.m, side);
    p.n_tiles = ceil_div(p.n, side);
    require(int64_t(p.m_tiles) * p.n_tiles * threads < (int64_t(1) << 31) && int64_t(p.splits) * p.batch < 65536,
            "too many workgroups");
    hipLaunchKernelGGL(kernel, dim3(unsigned(p.m_tiles) * p.n_tiles, unsigned(p.splits) * p.batch), threads, 0, d.stream, p, e);
    HIP_CHECK(hipGetLastError());
}

// p: the operands, sizes and batch; its cut is made here.
template <class T, bool AK, bool BK, class E>
void launch_product(Device& d, ProductArgs p, const E& e) {
    if (!p.m || !p.n || !p.batch) return;
    const ProductCut c = cut_product(d.compute_units, p.batch, p.m, p.n, int64_t(p.k) * p.planes.count, sizeof(T), p.a.wide && p.b.wide);
    const int deep = std::max(1, ceil_div(p.k, kDepth<T>));
    p.span = ceil_div(deep, std::min(c.splits, deep));
    p.splits = ceil_div(deep, p.span);
    if (!p.a.wide || !p.b.wide) launch_tiles(d, product_k<T, AK, BK, 64, 32, 2, true, E>, 64, 256, p, e);
    else if (c.side == 64) launch_tiles(d, product_k<T, AK, BK, 64, 32, 2, false, E>, 64, 256, p, e);
    else if (c.side == 128) launch_tiles(d, product_k<T, AK, BK, 128, 64, 2, false, E>, 128, 256, p, e);
    else if constexpr (sizeof(T) == 2) launch_tiles(d, product_large_k<T, AK, BK, E>, 256, 512, p, e);
    if (p.splits > 1) {
        const int64_t lanes = int64_t(p.batch) * p.m * ((p.n + 7) / 8);
        hipLaunchKernelGGL((product_join_k<E>), unsigned((lanes + 255) / 256), 256, 0, d.stream, p, e);
        HIP_CHECK(hipGetLastError());
    }
}

}  // namespace
}  // namespace cpde
