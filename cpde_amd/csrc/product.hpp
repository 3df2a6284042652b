// Matrix products on tiles: C[m][n] = sum over k of A(m, k) B(n, k), each operand with
// either of its axes contiguous, and an epilogue on rows of C before they are stored.
#pragma once
#include "sequence.hpp"

namespace cpde {
namespace {

// A matrix of a product: `stride` bytes from row to row.  Rows are m (or n) where k is
// contiguous, and k where m (or n) is.  It may be one of a batch, `batch` bytes apart.
// wide: its rows are read in whole 16-byte chunks, and its stride leaves a tile's offsets in
// 31 bits.
struct Operand {
    const char* data;
    int64_t stride, batch;
    int wide;
};
struct ProductArgs {
    Operand a, b;
    int m, n, k, batch;
    int symmetric;     // C is symmetric: tiles on and below its diagonal, mirrored as they are stored
    int m_tiles, n_tiles;
    int splits, span;  // of the inner axis, and a split's tiles of it
    float* part;       // [split][batch][m][n, to whole eights] where there are several
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

// A fragment of floats as three of bf16 values whose sums they are, exactly: the leading
// 8 of the 24 bits, the next 8 and the rest, cut off by masks (rounding each took a third
// more instructions).  Six of the nine products of two such sums leave out 2^-21 of the
// factors' at most and take 192 cycles where the float instruction takes 512; what is
// split is shared by the products of a wave's tile.
struct Split {
    Frag<bf16> part[3];
};
__device__ inline Split split(Frag<float> x) {
    Split s;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        vec<uint32_t, 4> two;
#pragma unroll
        for (int j = 0; j < 4; ++j)  // the upper halves of two floats
            two[j] = __builtin_amdgcn_perm(__float_as_uint(x[2 * j + 1]), __float_as_uint(x[2 * j]), 0x07060302u);
        s.part[i] = __builtin_bit_cast(Frag<bf16>, two);
        if (i < 2)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] -= __uint_as_float(__float_as_uint(x[j]) & 0xffff0000u);
    }
    return s;
}
__device__ inline Acc multiply(const Split& a, const Split& b, Acc c) {
    c = multiply(a.part[2], b.part[0], c);  // (the smallest first)
    c = multiply(a.part[0], b.part[2], c);
    c = multiply(a.part[1], b.part[1], c);
    c = multiply(a.part[1], b.part[0], c);
    c = multiply(a.part[0], b.part[1], c);
    return multiply(a.part[0], b.part[0], c);
}
// A fragment as it is multiplied.
template <bool Exact, class F>
__device__ inline auto part(const F& f) {
    if constexpr (std::is_same_v<F, Frag<float>> && !Exact) return split(f);
    else return f;
}

// A sum of two f16 values, 22 bits together where the second is one of the type's normal values
// (smaller sums are off by 2^-25 at most).  Matrices of them hold 32 first parts and then
// the 32 second ones, and so on, in rows of whole such groups.  Three of the four products
// are exact to 2^-21 of the factors'.
struct Pair {
    _Float16 part[2];
};
struct PairFragment {
    Frag<_Float16> part[2];
};
__device__ inline Acc multiply(const PairFragment& a, const PairFragment& b, Acc c) {
    c = multiply(a.part[1], b.part[0], c);
    c = multiply(a.part[0], b.part[1], c);
    return multiply(a.part[0], b.part[0], c);
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
        if (std::is_same_v<T, float>) return (((row >> 3) & 1) << 3) & (kChunks - 1);
        return ((row & 3) << 2) & (kChunks - 1);
    }
    // Of 32 columns from a chunk on: sixteen lanes read four k-rows of sixteen values (four lanes a
    // row) and get them back transposed, a column each.
    template <class V>
    __device__ static Frag<V> transposed(const char* tile, int first, int s, int lane) {
        const int row = 16 * s + 8 * (lane >> 5) + ((lane & 15) >> 2), chunk = first + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4* at;
        // (four rows on, the turn is the same)
        const char* p = tile + row * kRowBytes + ((chunk ^ turn(row)) << 4) + (lane & 1) * 8;
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(p));
        const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(p + 4 * kRowBytes));
        return __builtin_bit_cast(Frag<V>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    // Fragment of rows 32 block + lane % 32, inner indices 16 s + 8 (lane / 32) + j.
    __device__ static auto fragment(const char* tile, int block, int s, int lane) {
        const int half = lane >> 5;
        if constexpr (std::is_same_v<T, Pair>) {
            PairFragment f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if constexpr (K) {
                    const int row = 32 * block + (lane & 31);
                    f.part[i] = *reinterpret_cast<const Frag<_Float16>*>(tile + row * kRowBytes + (((4 * i + 2 * s + half) ^ turn(row)) << 4));
                } else {
                    f.part[i] = transposed<_Float16>(tile, 8 * block + 4 * i, s, lane);
                }
            return f;
        } else if constexpr (K && sizeof(T) == 2) {
            const int row = 32 * block + (lane & 31);
            return *reinterpret_cast<const Frag<T>*>(tile + row * kRowBytes + (((2 * s + half) ^ turn(row)) << 4));
        } else if constexpr (K) {
            const int row = 32 * block + (lane & 31);
            const char* p = tile + row * kRowBytes;
            const auto lo = *reinterpret_cast<const vec<T, 4>*>(p + (((4 * s + 2 * half) ^ turn(row)) << 4));
            const auto hi = *reinterpret_cast<const vec<T, 4>*>(p + (((4 * s + 2 * half + 1) ^ turn(row)) << 4));
            return Frag<T>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else if constexpr (sizeof(T) == 2) {
            return transposed<T>(tile, 4 * block, s, lane);
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
    uint32_t low, high;  // the address of the next tile, the same in every lane
    int64_t stride;
    int rows, left;      // rows (columns) from there on, inner indices
    bool ample;          // a row in memory is a chunk at least

    __device__ void start(const Operand& o, int batch, int first, int all, int k, int t) {
        const uint64_t at = reinterpret_cast<uint64_t>(o.data) + batch * o.batch +
                            (K ? int64_t(first) * o.stride : int64_t(first) * int64_t(sizeof(T))) + t * step(o.stride);
        low = uniform(int(uint32_t(at)));
        high = uniform(int(uint32_t(at >> 32)));
        stride = o.stride;
        rows = all - first;
        ample = (K ? k : all) >= kChunk;
        left = k - t * kDeep;
    }
    __device__ static int64_t step(int64_t stride) { return K ? kTileBytes : kDeep * stride; }  // from tile to tile
    __device__ uint64_t base() const { return (uint64_t(high) << 32) | low; }
    __device__ __attribute__((always_inline)) void next() {
        const uint64_t at = base() + step(stride);
        low = uint32_t(at);
        high = uint32_t(at >> 32);
        left -= kDeep;
    }
    // Byte offset of a lane's chunk i of a tile with `left` inner indices.  Rows past the
    // last repeat it (their results are not stored); inner indices past the end are zeros.
    __device__ uint32_t place(int i, int left) const {
        const int slot = i * Threads + threadIdx.x % Threads, row = slot / kChunks, chunk = (slot % kChunks) ^ turn(row);
        // (a group of pairs is eight chunks, four of either part)
        constexpr bool pairs = std::is_same_v<T, Pair>;
        if (K) return (pairs ? 8 * (chunk & 3) : chunk * kChunk) < left ? uint32_t(min(row, rows - 1)) * uint32_t(stride) + (chunk << 4) : kNone;
        const int chunks = pairs ? (rows + 31) / 32 * 8 : (rows + kChunk - 1) / kChunk;
        return row < left ? uint32_t(row) * uint32_t(stride) + (min(chunk, chunks - 1) << 4) : kNone;
    }
    __device__ void places(uint32_t (&offset)[kSteps]) const {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) offset[i] = place(i, kDeep);
    }
    // From memory to LDS without registers, for operands of whole 16-byte chunks.  The
    // loads have arrived after loads_arrived() and a barrier.
    __device__ __attribute__((always_inline)) void load(char* tile, const uint32_t (&offset)[kSteps], int wave) const {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's compiler does not know a buffer's type)
        const auto buffer = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base()), 0, 0x7ffffff0, 0x00020000);
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
    // Through registers, for any other, by 16-byte loads of any alignment, all under way at
    // once.  16-bit chunks over the end of a row are loaded as far ahead as they go over it, and
    // moved back (gradients of 8,192 rows, 255 -> 255: 44 us; value by value 110).  Floats there,
    // and rows shorter than a chunk, go value by value (the same in floats: 53 us; moved 62).
    using Chunk = vec<std::conditional_t<std::is_same_v<T, Pair>, float, T>, kChunk>;
    using Held = Chunk[kSteps];
    // Of eight 16-bit values those from `by` (0 to 8) on, then zeros.
    __device__ static Chunk moved(Chunk chunk, int by) {
        vec<uint32_t, 4> w = __builtin_bit_cast(decltype(w), chunk);
        const vec<uint32_t, 4> half = {__builtin_amdgcn_alignbit(w[1], w[0], 16), __builtin_amdgcn_alignbit(w[2], w[1], 16),
                                       __builtin_amdgcn_alignbit(w[3], w[2], 16), w[3] >> 16};
        w = by & 1 ? half : w;
        w = by & 2 ? vec<uint32_t, 4>{w[1], w[2], w[3], 0} : w;
        w = by & 4 ? vec<uint32_t, 4>{w[2], w[3], 0, 0} : w;
        w = by & 8 ? vec<uint32_t, 4>{0, 0, 0, 0} : w;
        return __builtin_bit_cast(Chunk, w);
    }
    __device__ __attribute__((always_inline)) void fetch(Held& held) const {
        if constexpr (std::is_arithmetic_v<T> || sizeof(T) == 2) {
            const auto row_of = [&](int row) __attribute__((always_inline)) { return reinterpret_cast<const T*>(base() + int64_t(row) * stride); };
            const int end = K ? left : rows, last = K ? rows - 1 : left - 1;  // of rows from here on, and the last row
            const auto place_of = [&](int i, int& row, int& first) __attribute__((always_inline)) {
                const int slot = i * Threads + threadIdx.x % Threads;
                row = slot / kChunks;
                first = ((slot % kChunks) ^ turn(row)) * kChunk;
            };
            int row, first;
            if (left >= kDeep && (K || rows >= N)) {
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    place_of(i, row, first);
                    __builtin_memcpy(&held[i], row_of(min(row, last)) + first, 16);
                }
            } else if (sizeof(T) == 2 && ample) {
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    place_of(i, row, first);
                    __builtin_memcpy(&held[i], row_of(min(row, last)) + min(first, end - kChunk), 16);
                }
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    place_of(i, row, first);
                    // (!K: inner indices past the end are rows of zeros)
                    held[i] = moved(held[i], !K && row > last ? kChunk : min(max(0, first - (end - kChunk)), kChunk));
                }
            } else {
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    place_of(i, row, first);
                    const T* p = row_of(min(row, last)) + first;
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) held[i][j] = first + j < end && (K || row <= last) ? p[j] : T(0.f);
                }
            }
        }
    }
    __device__ __attribute__((always_inline)) void put(char* tile, const Held& held) const {
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            *reinterpret_cast<Chunk*>(tile + (i * Threads + threadIdx.x % Threads) * 16) = held[i];
    }
};

__device__ inline void loads_arrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0), the other counters open

// All but the last N loads have arrived (the other counters stay open).
template <int N>
__device__ inline void arrived_but() { __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14)); }

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

// Where a split's sums of row m from column n on stand: rows of whole eights.
__device__ inline int64_t part_at(const ProductArgs& p, int split, int64_t batch, int64_t m, int n) {
    return ((int64_t(split) * p.batch + batch) * p.m + m) * ((p.n + 7) & ~7) + n;
}

// The tiles on and below the diagonal, row by row.
__device__ inline void triangle_of(int at, int& tm, int& tn) {
    tm = int((sqrtf(8.f * at + 1.f) - 1.f) * 0.5f);
    while (tm * (tm + 1) / 2 > at) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= at) ++tm;
    tn = at - tm * (tm + 1) / 2;
}

// Up to eight neighbouring values of a row, as floats; eight by 16-byte accesses of any
// alignment.
template <class T>
__device__ inline void read8(float (&v)[8], const T* p, int count) {
    if (count == 8) {
        vec<T, 8> in;
        __builtin_memcpy(&in, p, sizeof(in));
        const auto wide = __builtin_convertvector(in, vec<float, 8>);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = wide[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < count ? float(p[j]) : 0.f;
    }
}
template <class T>
__device__ inline void write8(T* p, const float (&v)[8], int count) {
    if (count == 8) {
        vec<float, 8> wide;
#pragma unroll
        for (int j = 0; j < 8; ++j) wide[j] = v[j];
        const vec<T, 8> out = __builtin_convertvector(wide, vec<T, 8>);
        __builtin_memcpy(p, &out, sizeof(out));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) p[j] = T(v[j]);
    }
}

// What the kernels of products share: C's tile [BM][BN] by waves of [WM][WN] each, two
// tiles of either operand in LDS.
template <class T, bool AK, bool BK, int BM, int BN, int WM, int WN, int Stages = 2, bool Exact = false>
struct Tiles {
    static constexpr int kThreads = (BM / WM) * (BN / WN) * 64, kMB = WM / 32, kNB = WN / 32, kS = kDepth<T> / 16;
    using A = TileSide<T, AK, BM, kThreads>;
    using B = TileSide<T, BK, BN, kThreads>;
    static constexpr int kPitch = WN + 4, kStage = 32 * kPitch * 4;  // a wave's rows of C on their way out
    static constexpr int kTile = A::kBytes + B::kBytes, kOut = kThreads / 64 * kStage;
    static constexpr int kLds = Stages * kTile > kOut ? Stages * kTile : kOut;
    static constexpr int kLoads = A::kSteps + B::kSteps;  // of a tile, by each lane

    using P = decltype(part<Exact>(A::fragment(nullptr, 0, 0, 0)));

    A a;
    B b;
    uint32_t a_offset[A::kSteps], b_offset[B::kSteps];
    int lane, wave, wm, wn, split, batch, m0, n0, steps, mirrored;
    Acc acc[kMB][kNB];

    __device__ __attribute__((always_inline)) void start(const ProductArgs& p) {
        lane = threadIdx.x & 63;
        wave = uniform(threadIdx.x >> 6);
        wm = wave % (BM / WM);
        wn = wave / (BM / WM);
        split = blockIdx.y % p.splits;
        batch = blockIdx.y / p.splits;
        int tm, tn;
        if (p.symmetric) triangle_of(blockIdx.x, tm, tn);
        else tile_of(blockIdx.x, p.m_tiles * p.n_tiles, p.m_tiles, p.n_tiles, tm, tn);
        mirrored = p.symmetric && tm != tn;
        m0 = tm * BM;
        n0 = tn * BN;
        const int t = split * p.span;
        a.start(p.a, batch, m0, p.m, p.k, t);
        b.start(p.b, batch, n0, p.n, p.k, t);
        a.places(a_offset);
        b.places(b_offset);
        steps = max(0, min((p.k + kDepth<T> - 1) / kDepth<T> - t, p.span));
#pragma unroll
        for (int i = 0; i < kMB; ++i)
#pragma unroll
            for (int j = 0; j < kNB; ++j) acc[i][j] = Acc{};
    }
    // The next tile's loads.
    __device__ __attribute__((always_inline)) void load(char* tile) {
        a.load(tile, a_offset, wave);
        b.load(tile + A::kBytes, b_offset, wave);
        a.next();
        b.next();
    }
    __device__ __attribute__((always_inline)) void fragments(const char* tile, int s, P (&fa)[kMB], P (&fb)[kNB]) const {
#pragma unroll
        for (int i = 0; i < kMB; ++i) fa[i] = part<Exact>(A::fragment(tile, wm * kMB + i, s, lane));
#pragma unroll
        for (int i = 0; i < kNB; ++i) fb[i] = part<Exact>(B::fragment(tile + A::kBytes, wn * kNB + i, s, lane));
    }
    __device__ __attribute__((always_inline)) void products(const P (&fa)[kMB], const P (&fb)[kNB]) {
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
        const int half = lane >> 5, column = (lane % kLanes) * 8, n = n0 + wn * WN + column;
        const auto columns = e.columns(batch, n, min(8, p.n - n));
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
                const int row = r * kAtOnce + lane / kLanes, m = m0 + wm * WM + 32 * i + row;
                float v[8];
                *reinterpret_cast<Quad*>(v) = *reinterpret_cast<const Quad*>(stage + row * kPitch + column);
                *reinterpret_cast<Quad*>(v + 4) = *reinterpret_cast<const Quad*>(stage + row * kPitch + column + 4);
                if (m >= p.m || n >= p.n) continue;
                if (p.splits > 1)
                    write8(p.part + part_at(p, split, batch, m, n), v, 8);
                else
                    e.row(columns, batch, m, n, min(8, p.n - n), v);
            }
            if constexpr (Epilogue::kSymmetric) {
                // the same with rows and columns exchanged: eight rows of a column a lane
                if (mirrored && p.splits == 1)
#pragma unroll
                    for (int r = 0; r < WN / 16; ++r) {
                        const int to = r * 16 + lane / 4, from = 8 * (lane % 4);
                        const int m = n0 + wn * WN + to, n = m0 + wm * WM + 32 * i + from;
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = stage[(from + j) * kPitch + to];
                        if (m < p.n && n < p.m) e.row(e.columns(batch, n, min(8, p.m - n)), batch, m, n, min(8, p.m - n), v);
                    }
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
};

// The loads of the next Stages - 1 tiles are under way while one is multiplied.  Any:
// operands of any alignment.
template <class T, bool AK, bool BK, int Side, int WM, int WN, int Stages, int PerSimd, bool Any, class Epilogue>
__global__ __launch_bounds__((Side / WM) * (Side / WN) * 64, PerSimd) void product_k(ProductArgs p, Epilogue e) {
    using C = Tiles<T, AK, BK, Side, Side, WM, WN, Stages, (Side < 128)>;
    __shared__ __align__(16) char lds[C::kLds];
    C c;
    c.start(p);
    // (the tiles read and written do not overlap, which the compiler has to know so as
    // not to wait for the loads under way before it reads)
    const auto step = [&](const char* __restrict__ tile, auto load) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < C::kS; ++s) {
            typename C::P fa[C::kMB], fb[C::kNB];
            c.fragments(tile, s, fa, fb);
            if (s == 0) load();
            c.products(fa, fb);
        }
    };
    if constexpr (Any) {
        // (what goes through registers is under way while the tile before is multiplied)
        typename C::A::Held ha;
        typename C::B::Held hb;
        const auto fetch = [&]() __attribute__((always_inline)) {
            if (!p.a.wide) {
                c.a.fetch(ha);
                c.a.next();
            }
            if (!p.b.wide) {
                c.b.fetch(hb);
                c.b.next();
            }
        };
        if (c.steps > 0) fetch();
        for (int i = 0; i < c.steps; ++i) {
            if (p.a.wide) {
                c.a.load(lds, c.a_offset, c.wave);
                c.a.next();
            } else {
                c.a.put(lds, ha);
            }
            if (p.b.wide) {
                c.b.load(lds + C::A::kBytes, c.b_offset, c.wave);
                c.b.next();
            } else {
                c.b.put(lds + C::A::kBytes, hb);
            }
            loads_arrived();
            __syncthreads();
            if (i + 1 < c.steps) fetch();
            step(lds, [] {});
            __syncthreads();
        }
    } else {
        int to = 0;  // the place of the next loads
        const auto load = [&](int i) __attribute__((always_inline)) {
            if (i < c.steps) c.load(lds + to * C::kTile);
            to = to + 1 == Stages ? 0 : to + 1;
        };
        int from = 0;
#pragma unroll
        for (int i = 0; i < Stages - 1; ++i) load(i);
        for (int i = 0; i < c.steps; ++i) {
            if (c.steps - i >= Stages - 1) arrived_but<(Stages - 2) * C::kLoads>();
            else loads_arrived();
            // (every wave's reads of the tile before, whose place is written next, are done)
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
            asm volatile("s_barrier" ::: "memory");
            step(lds + from * C::kTile, [&]() __attribute__((always_inline)) { load(i + Stages - 1); });
            from = from + 1 == Stages ? 0 : from + 1;
        }
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
    if (c.steps) c.load(lds);
    loads_arrived();
    __syncthreads();
    if (second) barrier();
    for (int i = 0; i < c.steps; ++i) {
        const char* tile = lds + (i & 1) * C::kTile;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            constexpr int kSteps = C::kS / 2;
            typename C::P fa[kSteps][C::kMB], fb[kSteps][C::kNB];
#pragma unroll
            for (int s = 0; s < kSteps; ++s) c.fragments(tile, kSteps * part + s, fa[s], fb[s]);
            __builtin_amdgcn_sched_barrier(0);
            if (part == 0 && i + 1 < c.steps) c.load(lds + ((i + 1) & 1) * C::kTile);
            if (part == 1 && second) loads_arrived();
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the reads
            barrier();
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) c.products(fa[s], fb[s]);
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

// Small products and few rows: a workgroup makes a tile of 32 x 32, its waves sharing the
// inner axis, each with tiles of its own in LDS, two at a time and no barrier until
// their sums are joined.  Bound: the latency of a launch and of a round or two of loads; with
// few rows and a large matrix, HBM (16 rows, 2048 -> 8192, bf16: 34 MB in 7.9 us, 4.3 TB/s; 11.8 by
// split 64 x 64 tiles and a join; fragments straight from memory, 32 bytes a row, 11.3).
template <class T, bool AK, bool BK, bool Any, class Epilogue>
__global__ __launch_bounds__(512) void product_run_k(ProductArgs p, Epilogue e) {
    extern __shared__ __align__(16) char lds[];  // [wave][2][A, B], then [wave][32][36] sums
    using A = TileSide<T, AK, 32, 64>;
    using B = TileSide<T, BK, 32, 64>;
    constexpr int kTile = A::kBytes + B::kBytes, kPitch = 36;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), waves = blockDim.x / 64, half = lane >> 5;
    int tm, tn;
    tile_of(blockIdx.x, p.m_tiles * p.n_tiles, p.m_tiles, p.n_tiles, tm, tn);
    const int m0 = tm * 32, n0 = tn * 32, batch = blockIdx.y;
    const int deep = (p.k + A::kDeep - 1) / A::kDeep, share = (deep + waves - 1) / waves;
    const int first = wave * share, steps = min(deep - first, share);
    A a;
    B b;
    a.start(p.a, batch, m0, p.m, p.k, first);
    b.start(p.b, batch, n0, p.n, p.k, first);
    uint32_t a_offset[A::kSteps], b_offset[B::kSteps];
    a.places(a_offset);
    b.places(b_offset);
    char* mine = lds + wave * 2 * kTile;
    // (what goes through registers is put in LDS when the tile before has been multiplied)
    typename A::Held ha;
    typename B::Held hb;
    const auto load = [&](int i) __attribute__((always_inline)) {
        char* tile = mine + (i & 1) * kTile;
        if (Any && !p.a.wide) a.fetch(ha);
        else a.load(tile, a_offset, 0);
        if (Any && !p.b.wide) b.fetch(hb);
        else b.load(tile + A::kBytes, b_offset, 0);
        a.next();
        b.next();
    };
    const auto put = [&](int i) __attribute__((always_inline)) {
        char* tile = mine + (i & 1) * kTile;
        if (!p.a.wide) a.put(tile, ha);
        if (!p.b.wide) b.put(tile + A::kBytes, hb);
    };
    Acc acc = {};
    if (steps > 0) {
        load(0);
        if (Any) put(0);
    }
    for (int i = 0; i < steps; ++i) {
        if (Any && (p.a.wide || p.b.wide)) loads_arrived();
        if (i + 1 < steps) load(i + 1);
        if (!Any) {
            if (i + 1 < steps) arrived_but<A::kSteps + B::kSteps>();
            else loads_arrived();
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): stores to LDS, and the reads of the tile before
        asm volatile("" ::: "memory");
        const char* tile = mine + (i & 1) * kTile;
#pragma unroll
        for (int s = 0; s < kDepth<T> / 16; ++s)
            acc = multiply(B::fragment(tile + A::kBytes, 0, s, lane), A::fragment(tile, 0, s, lane), acc);
        // (the next loads write where these reads were)
        __builtin_amdgcn_s_waitcnt(0xc07f);
        asm volatile("" ::: "memory");
        if (Any && i + 1 < steps) put(i + 1);
    }
    __syncthreads();
    float* sums = reinterpret_cast<float*>(lds);
    float* to = sums + (wave * 32 + (lane & 31)) * kPitch;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const Quad v = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
        *reinterpret_cast<Quad*>(to + 8 * g + 4 * half) = v;
    }
    __syncthreads();
    // eight columns of a row a lane
    for (int at = threadIdx.x; at < 128; at += blockDim.x) {
        const int row = at / 4, column = at % 4 * 8;
        float v[8] = {};
        for (int w = 0; w < waves; ++w) {
            const float* from = sums + (w * 32 + row) * kPitch + column;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += from[j];
        }
        const int n = n0 + column, count = min(8, p.n - n);
        if (m0 + row < p.m && n < p.n) e.row(e.columns(batch, n, count), batch, m0 + row, n, count, v);
    }
}
template <class T>
constexpr size_t kRunBytes = 2 * 2 * 32 * kTileBytes;  // of LDS for each wave

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
        read8(one, p.part + part_at(p, s, 0, row, n), 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += one[j];
    }
    e.row(e.columns(batch, n, count), batch, int(row - int64_t(batch) * p.m), n, count, v);
}

// The same of a symmetric product: 64 x 64 on and below the diagonal a workgroup, stored
// twice.
template <class Epilogue>
__global__ __launch_bounds__(256) void product_join_symmetric_k(ProductArgs p, Epilogue e) {
    __shared__ float stage[64][65];
    int tm, tn;
    triangle_of(blockIdx.x, tm, tn);
    const int batch = blockIdx.y, row = threadIdx.x / 4, column = threadIdx.x % 4 * 16;
#pragma unroll
    for (int part = 0; part < 16; part += 8) {
        const int m = tm * 64 + row, n = tn * 64 + column + part, count = min(8, p.n - n);
        float v[8] = {};
        if (m < p.m && n < p.n) {
            for (int s = 0; s < p.splits; ++s) {
                float one[8];
                read8(one, p.part + part_at(p, s, batch, m, n), 8);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += one[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) stage[row][column + part + j] = v[j];
        if (m < p.m && n < p.n) e.row(e.columns(batch, n, count), batch, m, n, count, v);
    }
    __syncthreads();
    if (tm == tn) return;
#pragma unroll
    for (int part = 0; part < 16; part += 8) {
        const int m = tn * 64 + row, n = tm * 64 + column + part, count = min(8, p.m - n);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = stage[column + part + j][row];
        if (m < p.n && n < p.m) e.row(e.columns(batch, n, count), batch, m, n, count, v);
    }
}

// ---- on the host --------------------------------------------------------------------------
inline int ceil_div(int64_t a, int64_t b) { return int((a + b - 1) / b); }

// How a product is cut: the side of its tiles (32: product_run_k, of `waves` waves), and
// splits of its inner axis.
struct ProductCut {
    int side = 64, splits = 1, waves = 4;
};
constexpr int kMostSplits = 32;
constexpr int64_t kPartTiles = 4;  // 128 x 128 tiles of partial sums a unit, at most

// By the times that the kernels take (microseconds, 256 CUs), measured with 128 to 1,024
// workgroups and inner axes of 256 to 4,096: what a launch takes with its first loads
// and its last stores, and a tile of the inner axis with one and with several
// workgroups a CU.
struct ProductTime {
    int side;
    double start, alone, shared;
};
constexpr ProductTime kTimes16[] = {{64, 3.8, 0.30, 0.195}, {128, 4.2, 0.62, 0.47}, {256, 11.5, 1.50, 1.50}};
constexpr ProductTime kTimes32[] = {{64, 4.5, 0.65, 0.53}, {128, 8.0, 1.55, 1.43}, {256, 14.0, 4.7, 4.7}};
constexpr ProductTime kTimesPair[] = {{64, 4.0, 0.40, 0.27}, {128, 5.0, 0.95, 0.75}, {256, 12.0, 2.2, 2.2}};
template <class T>
ProductCut cut_product(int compute_units, int64_t batch, int64_t m, int64_t n, int64_t k, bool wide, bool symmetric) {
    constexpr int size = sizeof(T);
    ProductCut best;
    double least = 1e30;
    const int64_t deep = std::max<int64_t>(1, (k + kTileBytes / size - 1) / (kTileBytes / size));
    const auto consider = [&](const ProductTime& t) {
        const int64_t rows = ceil_div(m, t.side), tiles = batch * (symmetric ? rows * (rows + 1) / 2 : rows * ceil_div(n, t.side));
        for (int splits = 1; splits <= kMostSplits && (splits == 1 || (splits * 2 <= deep && t.side < 256)); ++splits) {
            if (splits > 1 && splits * batch * m * ((n + 7) / 8 * 8) > kPartTiles * compute_units * 128 * 128) break;
            const int64_t each = (tiles * splits + compute_units - 1) / compute_units;
            double time = t.start + double((deep + splits - 1) / splits) * (each == 1 ? t.alone : std::max(t.alone, each * t.shared));
            if (splits > 1) time += 3.5 + double(batch) * m * n * splits * 8 / 4e6;
            if (time < least) {
                least = time;
                best.side = t.side;
                best.splits = splits;
            }
        }
    };
    const auto consider_all = [&](const auto& times) {
        for (const auto& t : times)
            if (wide || t.side == 64) consider(t);
    };
    if constexpr (std::is_same_v<T, Pair>) consider_all(kTimesPair);
    else if constexpr (size == 2) consider_all(kTimes16);
    else consider_all(kTimes32);
    // a workgroup of 32 x 32, one or two on a CU at once
    const int64_t tiles = batch * ceil_div(m, 32) * int64_t(ceil_div(n, 32));
    if (tiles <= 2 * compute_units) {
        const int waves = int(std::min<int64_t>(tiles <= compute_units ? 8 : 4, deep));
        const double time = 3.6 + double((deep + waves - 1) / waves) * (size == 2 ? 0.5 : 0.8);
        if (time < least) {
            best.side = 32;
            best.splits = 1;
            best.waves = waves;
        }
    }
    return best;
}
// Floats of ProductArgs::part that no call with up to `m` rows passes.
inline size_t product_part(int compute_units, int64_t batch, int64_t m, int64_t n) {
    return size_t(std::min<int64_t>(kPartTiles * compute_units * 128 * 128, kMostSplits * batch * m * ((n + 7) / 8 * 8)));
}

// An operand of rows of `columns` values of `size` bytes.  (A tile of 256 rows 2^22 bytes apart
// ends within 2^31 of its start.)
inline Operand product_operand(const void* data, int64_t stride, int64_t columns, size_t size) {
    Operand o{};
    o.data = static_cast<const char*>(data);
    o.stride = stride * int64_t(size);
    o.wide = wide(data, stride, size) && columns * size % 16 == 0 && o.stride <= (int64_t(1) << 22);
    return o;
}

// A product as it is launched: with its cut.
struct Product {
    ProductArgs args;
    ProductCut cut;
    bool wide;
    bool empty() const { return !args.m || !args.n || !args.batch; }
};
// Columns of a wave's part of a 128 x 128 tile: eight waves, or four where a fragment costs more:
// floats' splits (1,024 tiles, k = 1024: 185 us for 199), transposing reads of both operands (4096 x
// 2048, k = 8192, bf16: 133 for 156; of neither, 128 tiles, k = 1024: 13.7, and 11.9 by eight)
template <class T, bool AK, bool BK>
constexpr int kWave128 = std::is_same_v<T, float> || (!AK && !BK) ? 64 : 32;

// p: the operands, sizes and batch.  Its cut is made here, and a launch of too many workgroups
// refused, so that a call of several launches can cut all of them before its first one.
template <class T, bool AK, bool BK>
Product cut_for(const Device& d, ProductArgs p) {
    Product q{p, {}, p.a.wide && p.b.wide};
    if (q.empty()) return q;
    const ProductCut c = q.cut = cut_product<T>(d.compute_units, p.batch, p.m, p.n, p.k, q.wide, p.symmetric);
    const int deep = std::max(1, ceil_div(p.k, kDepth<T>));
    p.span = ceil_div(deep, std::min(c.splits, deep));
    p.splits = ceil_div(deep, p.span);
    if (c.side == 32) p.symmetric = 0;  // (whole tiles of both halves)
    p.m_tiles = ceil_div(p.m, c.side);
    p.n_tiles = ceil_div(p.n, c.side);
    q.args = p;
    const int threads = c.side == 32 ? 64 * c.waves : c.side == 64 ? 256 : c.side == 128 ? 256 * 64 / kWave128<T, AK, BK> : 512;
    const int64_t tiles = p.symmetric ? int64_t(p.m_tiles) * (p.m_tiles + 1) / 2 : int64_t(p.m_tiles) * p.n_tiles;
    require(tiles * threads < (int64_t(1) << 31) && int64_t(p.splits) * p.batch < 65536, "too many workgroups");
    return q;
}

// A launch of one of the kernels of tiles.
template <class K, class E>
void launch_tiles(Device& d, K kernel, int threads, const ProductArgs& p, const E& e, size_t lds = 0) {
    const int tiles = p.symmetric ? p.m_tiles * (p.m_tiles + 1) / 2 : p.m_tiles * p.n_tiles;
    hipLaunchKernelGGL(kernel, dim3(unsigned(tiles), unsigned(p.splits) * p.batch), threads, lds, d.stream, p, e);
    HIP_CHECK(hipGetLastError());
}

template <class T, bool AK, bool BK, class E>
void launch_product(Device& d, const Product& q, const E& e) {
    if (q.empty()) return;
    constexpr bool kAny = E::kAny;  // (whether operands may be of any alignment)
    const ProductArgs& p = q.args;
    const ProductCut& c = q.cut;
    require(q.wide || kAny, "operands of products are aligned");
    if (c.side == 32) {
        const size_t lds = c.waves * kRunBytes<T>;
        if (q.wide) {
            launch_tiles(d, product_run_k<T, AK, BK, false, E>, 64 * c.waves, p, e, lds);
        } else {
            if constexpr (kAny) launch_tiles(d, product_run_k<T, AK, BK, true, E>, 64 * c.waves, p, e, lds);
        }
    } else if (!q.wide) {
        if constexpr (kAny) launch_tiles(d, product_k<T, AK, BK, 64, 32, 32, 1, 2, true, E>, 256, p, e);
    } else if (c.side == 64) {
        launch_tiles(d, product_k<T, AK, BK, 64, 32, 32, 3, 2, false, E>, 256, p, e);
    } else if (c.side == 128) {
        constexpr int kWave = kWave128<T, AK, BK>;
        launch_tiles(d, product_k<T, AK, BK, 128, 64, kWave, 2, 128 / kWave, false, E>, 256 * 64 / kWave, p, e);
    } else {
        launch_tiles(d, product_large_k<T, AK, BK, E>, 512, p, e);
    }
    if (p.splits > 1) {
        if constexpr (E::kSymmetric)
            if (p.symmetric) {
                const int64_t rows = ceil_div(p.m, 64);
                hipLaunchKernelGGL((product_join_symmetric_k<E>), dim3(unsigned(rows * (rows + 1) / 2), unsigned(p.batch)), 256, 0,
                                   d.stream, p, e);
                HIP_CHECK(hipGetLastError());
                return;
            }
        const int64_t lanes = int64_t(p.batch) * p.m * ((p.n + 7) / 8);
        hipLaunchKernelGGL((product_join_k<E>), unsigned((lanes + 255) / 256), 256, 0, d.stream, p, e);
        HIP_CHECK(hipGetLastError());
    }
}
template <class T, bool AK, bool BK, class E>
void launch_product(Device& d, const ProductArgs& p, const E& e) {
    launch_product<T, AK, BK>(d, cut_for<T, AK, BK>(d, p), e);
}

}  // namespace
}  // namespace cpde
