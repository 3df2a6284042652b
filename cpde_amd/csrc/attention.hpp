// Attention: the kernels' arguments and their building blocks.
#pragma once
#include "sequence.hpp"

namespace cpde {

constexpr int kWaveRows = 32;      // query rows (or keys, in the keys' gradients) of a wave: one matrix tile's side
constexpr int kBlockRows = 128;    // of a workgroup of four waves
constexpr int kMaxHeadDim = 128;

// A tensor [batch][token][head][dim] with strides in elements.
struct HeadView {
    char* data;
    int64_t batch, token, head;
};

// Query rows of a key head are counted query by query, the heads of its group side
// by side: row r is query r / group of query head r % group.
struct AttentionArgs {
    HeadView q, k, v, out, dout, dq, dk, dv;
    float* lse;
    const int *query_lengths, *key_lengths;
    int pairs, kv_heads, group;  // pairs: batch entries x key heads
    int key_blocks;              // workgroups of the keys' gradients, the first of their launch
    int queries, keys, dim;
    int left, right;             // negative: unbounded
    int tiles, splits;           // of query rows
    int key_tiles, key_splits;   // of keys, in their gradients
    int span;                    // keys of a split of the vector kernel
    float scale, scale2;         // of the scores; the same times log2 e
    int wide_in, wide_out;       // 16-byte loads and stores
    float *part, *part_stats;    // [split][pair][row][dim], [split][pair][row][2]
    float* key_part;             // dk, then dv: [split][pair][key][dim] each
    float *row_lse, *row_delta;  // [batch][head][query]: lse (less kLift) over scale, dout.out
};

// Lengths of a batch entry.
__device__ inline int length_of(const int* lengths, int b, int most) {
    return lengths ? min(max(lengths[b], 0), most) : most;
}

// Keys [lo, hi) that query i of a batch entry sees, and queries that see key j.
struct Band {
    int ql, kl, left, right;
    __device__ Band(const AttentionArgs& a, int b)
        : ql(length_of(a.query_lengths, b, a.queries)), kl(length_of(a.key_lengths, b, a.keys)), left(a.left),
          right(a.right) {}
    __device__ int key_lo(int i) const { return left < 0 ? 0 : min(max(i + kl - ql - left, 0), kl); }
    __device__ int key_hi(int i) const { return right < 0 ? kl : max(min(i + kl - ql + right + 1, kl), 0); }
    __device__ int query_lo(int j) const { return right < 0 ? 0 : min(max(j - (kl - ql) - right, 0), ql); }
    __device__ int query_hi(int j) const { return left < 0 ? ql : max(min(j - (kl - ql) + left + 1, ql), 0); }
};

// Base-2 exponential and logarithm in one instruction each (relative error about
// 1e-7; results below the normal range are zeros).
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// ---- matrix tiles ---------------------------------------------------------------------
// A 32 x 32 product tile C = A B: lane l holds column l % 32 of C, at rows
// 8 g + 4 (l / 32) + j in element 4 g + j.  A fragment is 8 values along the inner
// axis, at 8 (l / 32) + j, of A's row or B's column l % 32; which inner index stands
// in which place is free as long as A and B agree.
typedef float Acc __attribute__((ext_vector_type(16)));
template <class T>
using Frag = vec<T, 8>;

__device__ inline Acc mma(Frag<bf16> a, Frag<bf16> b, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline Acc mma(Frag<_Float16> a, Frag<_Float16> b, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline Acc mma(Frag<float> a, Frag<float> b, Acc c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
// Rows 16 s .. 16 s + 15 of a tile's columns as the fragment of a second product
// that sums over those rows: a lane's own elements, in the order in which
// Tile::column reads the other operand.
template <class T>
__device__ inline Frag<T> as_fragment(const Acc& c, int s) {
    vec<float, 8> v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c[8 * s + j];
    return __builtin_convertvector(v, Frag<T>);
}

// A tile [rows][DP] in LDS, in 16-byte chunks whose place in the row is turned with
// the row's number: eight neighbouring rows' chunks of the same column (a row
// fragment) and four neighbouring rows' pairs of chunks (a transposed one) lie in
// different banks.
template <class T, int DP>
struct Tile {
    static constexpr int kChunks = DP * int(sizeof(T)) / 16, kRowBytes = DP * int(sizeof(T)), kChunk = 16 / sizeof(T);
    __device__ static int turn(int row) {
        if (kChunks % 8 == 0) return ((row & 3) << 1) | ((row >> 2) & 1);
        return (row & 2) | ((row >> 2) & 1);  // (two rows of 64 or 192 bytes already differ)
    }
    // Fragment of row `row`, inner indices the columns 16 s + 8 half + j.
    __device__ static Frag<T> row(const char* tile, int row, int s, int half) {
        const char* p = tile + row * kRowBytes;
        if constexpr (sizeof(T) == 2 && (kChunks & (kChunks - 1)) == 0) {
            // (the same place, by one exclusive or a fragment)
            const int at = (row * kRowBytes + ((half ^ turn(row)) << 4)) ^ (s << 5);
            return *reinterpret_cast<const Frag<T>*>(tile + at);
        } else if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const Frag<T>*>(p + (((2 * s + half) ^ turn(row)) << 4));
        } else {
            const auto lo = *reinterpret_cast<const vec<T, 4>*>(p + (((4 * s + 2 * half) ^ turn(row)) << 4));
            const auto hi = *reinterpret_cast<const vec<T, 4>*>(p + (((4 * s + 2 * half + 1) ^ turn(row)) << 4));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // Fragment of column 32 block + lane % 32, inner indices the rows
    // 16 s + 8 (j / 4) + 4 half + j % 4.
    __device__ static Frag<T> column(const char* tile, int block, int s, int lane) {
        const int half = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            // Sixteen lanes read four rows of sixteen values (four lanes a row) and
            // get them back transposed, a column each.
            const int row = 16 * s + 4 * half + ((lane & 15) >> 2);
            const int chunk = 4 * block + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
            const char* p = tile + row * kRowBytes + ((chunk ^ turn(row)) << 4) + (lane & 1) * 8;
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s4* at;
            const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(p));
            const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(p + 8 * kRowBytes));
            return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int column = 32 * block + (lane & 31);
            Frag<T> f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = 16 * s + 8 * (j / 4) + 4 * half + j % 4;
                f[j] = *reinterpret_cast<const T*>(tile + row * kRowBytes + (((column >> 2) ^ turn(row)) << 4) +
                                                   (column & 3) * 4);
            }
            return f;
        }
    }
};

// A number that the compiler takes for a new one each time: what is derived from it
// is computed where it is used, not kept in registers through a loop.
__device__ inline int fresh(int i) {
    asm volatile("" : "+v"(i));
    return i;
}

// The power of two by which a gradient's probabilities are larger (Fit).
template <class T>
constexpr int kLift = std::is_same_v<T, _Float16> ? 14 : 0;

// Brings ROWS rows of a tensor into a tile, 256 lanes.  Rows past `valid` repeat
// the last valid one (the caller hides them): memory past the lengths is not read.
template <class T, int DP, int ROWS>
struct TileLoader {
    using L = Tile<T, DP>;
    static constexpr int kSlots = ROWS * L::kChunks, kSteps = (kSlots + 255) / 256;
    // Where 256 slots are whole rows in eights, a lane's slots differ by whole rows:
    // one lane's offset and a step that is the same in every lane.
    static constexpr bool kRegular = 256 % (8 * L::kChunks) == 0;
    // f16's gradients of 128-wide keys have no registers for addresses held ready: a
    // spilled one, reloaded behind the loads under way, waits for them (2 x 4096 causal,
    // 16 heads on 4, training: 893 us, 807 with addresses made anew).
    static constexpr bool kAnew = kLift<T> != 0 && DP == 128 && ROWS == 32;
    static constexpr uint32_t kNone = ~0u;   // a column past the head's width
    uint32_t offset[kRegular ? 1 : kSteps];  // of a full tile
    int chunks;                              // that hold values
    int64_t stride;                          // bytes from row to row
    int dim;
    bool direct;

    __device__ void start(int64_t token, int dim_, bool wide) {
        stride = token * int64_t(sizeof(T));
        dim = dim_;
        chunks = dim / L::kChunk;
        direct = wide;
#pragma unroll
        for (int i = 0; i < (kRegular ? 1 : kSteps); ++i) {
            const int slot = i * 256 + threadIdx.x, row = slot / L::kChunks, chunk = (slot % L::kChunks) ^ L::turn(row);
            offset[i] = chunk < chunks ? uint32_t(row * uint32_t(stride)) + (chunk << 4) : kNone;
        }
    }
    // Columns past the head's width are zeros: written once where rows are loaded
    // directly, which leaves them alone.
    __device__ void clear(char* tile) const {
        if (direct && chunks < L::kChunks)
            for (int slot = threadIdx.x; slot < kSlots; slot += 256)
                *reinterpret_cast<u32x4*>(tile + slot * 16) = u32x4{0, 0, 0, 0};
    }
    // wave: this wave's number, the same in every lane.  The loads have arrived
    // after arrived() and a barrier.
    __device__ __attribute__((always_inline)) void load(char* tile, const char* base, int valid, int wave) const {
        const auto bring = [&](int i, const char* from) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                             (__attribute__((address_space(3))) void*)(tile + (i * 256 + wave * 64) * 16),
                                             16, 0, 0);
        };
        if (direct && valid >= ROWS) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                if (kSlots % 256 && i * 256 + wave * 64 >= kSlots) break;
                const uint32_t at = kAnew ? fresh(offset[kRegular ? 0 : i]) : offset[kRegular ? 0 : i];
                if (at != kNone) bring(i, base + (kRegular ? i * (256 / L::kChunks) * stride : 0) + at);
            }
        } else if (direct) {
            const int lane = fresh(threadIdx.x);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int slot = i * 256 + lane, row = slot / L::kChunks, chunk = (slot % L::kChunks) ^ L::turn(row);
                if (slot < kSlots && chunk < chunks) bring(i, base + int64_t(min(row, valid - 1)) * stride + chunk * 16);
            }
        } else {
            for (int slot = fresh(threadIdx.x); slot < kSlots; slot += 256) {
                const int row = slot / L::kChunks, column = ((slot % L::kChunks) ^ L::turn(row)) * L::kChunk;
                const T* p = reinterpret_cast<const T*>(base + int64_t(min(row, valid - 1)) * stride);
                vec<T, L::kChunk> v;
#pragma unroll
                for (int j = 0; j < L::kChunk; ++j) v[j] = column + j < dim ? p[column + j] : T(0.f);
                *reinterpret_cast<vec<T, L::kChunk>*>(tile + slot * 16) = v;
            }
        }
    }
};
// The same for one wave and a tile of its own: 64 lanes, ROWS rows.
template <class T, int DP, int ROWS>
struct WaveLoader {
    using L = Tile<T, DP>;
    static constexpr int kSteps = ROWS * L::kChunks / 64;
    static constexpr uint32_t kNone = ~0u;  // a column past the head's width
    uint32_t offset[kSteps];
    int chunks, dim;
    int64_t stride;
    bool direct;

    __device__ void start(int64_t token, int dim_, bool wide, int lane) {
        stride = token * int64_t(sizeof(T));
        dim = dim_;
        chunks = dim / L::kChunk;
        direct = wide;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int slot = i * 64 + lane, row = slot / L::kChunks, chunk = (slot % L::kChunks) ^ L::turn(row);
            offset[i] = chunk < chunks ? uint32_t(row * uint32_t(stride)) + (chunk << 4) : kNone;
        }
    }
    // Columns past the head's width: zeros.  Only the chunks that direct loads leave
    // alone are written, as nothing orders a wave's stores to LDS and its loads into it.
    __device__ void clear(char* tile, int lane) const {
        if (direct && chunks < L::kChunks)
            for (int slot = lane; slot < ROWS * L::kChunks; slot += 64)
                if (((slot % L::kChunks) ^ L::turn(slot / L::kChunks)) >= chunks)
                    *reinterpret_cast<u32x4*>(tile + slot * 16) = u32x4{0, 0, 0, 0};
    }
    // The loads have arrived after arrived().
    __device__ __attribute__((always_inline)) void load(char* tile, const char* base, int valid, int lane) const {
        const auto bring = [&](int i, const char* from) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                             (__attribute__((address_space(3))) void*)(tile + i * 1024), 16, 0, 0);
        };
        if (direct && valid >= ROWS) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
                if (offset[i] != kNone) bring(i, base + offset[i]);
            return;
        }
        for (int i = 0; i < kSteps; ++i) {
            const int slot = i * 64 + fresh(lane), row = slot / L::kChunks, chunk = (slot % L::kChunks) ^ L::turn(row);
            const char* from = base + int64_t(min(row, valid - 1)) * stride;
            if (direct) {
                if (chunk < chunks) bring(i, from + chunk * 16);
            } else {
                vec<T, L::kChunk> v;
#pragma unroll
                for (int j = 0; j < L::kChunk; ++j) {
                    const int column = chunk * L::kChunk + j;
                    v[j] = column < dim ? reinterpret_cast<const T*>(from)[column] : T(0.f);
                }
                *reinterpret_cast<vec<T, L::kChunk>*>(tile + slot * 16) = v;
            }
        }
    }
};

__device__ inline void arrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0), the other counters open

// A row's fragments straight from memory: inner indices the columns 16 s + 8 half + j,
// zeros past `dim`.
template <class T, int DP>
__device__ inline void load_fragments(Frag<T>* f, const T* row, int dim, int half, bool live, bool wide) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int at = 16 * s + 8 * half;
#pragma unroll
        for (int part = 0; part < 8; part += N) {
            vec<T, N> v = {};
            if (live) {
                if (wide) {
                    if (at + part < dim) v = *reinterpret_cast<const vec<T, N>*>(row + at + part);
                } else {
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        if (at + part + j < dim) v[j] = row[at + part + j];
                }
            }
#pragma unroll
            for (int j = 0; j < N; ++j) f[s][part + j] = v[j];
        }
    }
}

// A lane's column of a 32-row tile (rows are the head's columns from 32 block) times
// `by`, into one row of an output.
template <class T>
__device__ inline void store_column(T* row, const Acc& c, float by, int block, int half, int dim, bool wide) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int at = 32 * block + 8 * g + 4 * half;
        if (wide) {
            if (at < dim) {
                vec<float, 4> v = {c[4 * g] * by, c[4 * g + 1] * by, c[4 * g + 2] * by, c[4 * g + 3] * by};
                const auto out = __builtin_convertvector(v, vec<T, 4>);
                *reinterpret_cast<vec<T, 4>*>(row + at) = out;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j < dim) row[at + j] = T(c[4 * g + j] * by);
        }
    }
}

// Nothing in a lane's column: of a row or key without a part in the call, whose place in
// the products a NaN or infinity of the others' may have reached (0 x NaN).
template <int N>
__device__ inline void clear(Acc (&c)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = Acc{};
}
// Whether any query sees a key.
__device__ inline bool seen(const Band& band, int key) {
    return key < band.kl && band.query_lo(key) < band.query_hi(key);
}

// The same over the two halves of a wave: lane l and lane l ^ 32 hold one column.
__device__ inline float halves_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float halves_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Score gradients ds = p (dp - delta) of f16 tensors are rounded to f16, whose normal range
// ends at 2^-14 and 2^16, and are about the output's gradient over the number of keys.  So
// p, which is at most 1, comes 2^kLift times as large, and each column's ds (a key's, or a
// query row's) times a power of two of its own, `by`: as large as can be at the start, and
// down, with the column's sums so far, where its largest would pass 2^15, to leave that above
// 2^11.  Roundings are relative down to 2^-25 of the largest so far, and 2^-36 of it below.
// (bf16 and f32 need none of it.)
template <class T>
struct Fit {
    float by = 0x1p100f;
    template <int M>
    __device__ __attribute__((always_inline)) void operator()(Acc& ds, Acc (&sum)[M]) {
        if constexpr (kLift<T> != 0) {
            float top = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(ds[i]));
            top = halves_max(top);
            const bool grown = top * by > 0x1p15f;
            if (__any(grown)) {
                // 2^(11 - the exponent)
                const float next = grown ? __uint_as_float((265 - (__float_as_uint(top) >> 23)) << 23) : by;
                const float down = next / by;
                by = next;
#pragma unroll
                for (int d = 0; d < M; ++d) sum[d] *= down;
            }
            ds *= by;
        }
    }
    // What takes both factors, and p's alone, off again.
    __device__ float off() const { return kLift<T> ? __builtin_ldexpf(1.f, -kLift<T>) / by : 1.f; }
    __device__ static float p_off() { return kLift<T> ? __builtin_ldexpf(1.f, -kLift<T>) : 1.f; }
};

template <class T>
__device__ inline T* head_row(const HeadView& v, int b, int64_t token, int head) {
    return reinterpret_cast<T*>(v.data) + b * v.batch + token * v.token + head * v.head;
}

}  // namespace cpde
