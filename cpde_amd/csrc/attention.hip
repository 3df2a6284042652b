// Attention over sets and sequences, and its gradient.
#include <cmath>
#include <cstdio>
#include <initializer_list>

#include "attention.hpp"

namespace cpde {
namespace {

// How the launches of a shape are cut (cut_launches).
struct Cut {
    bool step = false, brief = false;  // the forward runs on the vector kernel, of 16 waves
    bool few = false;                  // on the kernel of 32 rows a workgroup
    bool few_gradient = false;         // the backward on the one of 32 keys or rows
    int rows = 0, row_tiles = 0, key_tiles = 0;
    int span = 0, forward = 1, query = 1, key = 1;                   // splits (of `span` keys on the first two)
    size_t stats = 0, part = 0, part_stats = 0, key_part = 0, floats = 0;  // of the workspace
};
// Query rows of a key head up to which the vector kernel serves.
constexpr int kStepRows = 2;

struct Attention {
    Device* dev = nullptr;
    cpde_attention_shape shape{};
    Cut cut;
    double seen = 0;  // visible pairs at the full lengths, over the batch and the query heads
    float* work = nullptr;
};

// Keys of a tile of the forward and of the queries' gradients.
template <class T>
constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;
// Queries of a tile of the keys' gradients.
constexpr int kQueries = 32;
// Workgroups a CU's registers have to hold.
template <class T, int DP>
constexpr int kGroups = DP * sizeof(T) <= 256 ? 2 : 1;

// ---- forward --------------------------------------------------------------------------
// One pass over the keys with a running maximum and sum.  Scores are computed
// transposed (keys x queries), so that a lane holds 16 of every 32 keys of ONE
// query: its maximum, sum and rescaling are its own, but for one exchange with lane
// ^ 32, and its probabilities are, in place, the fragment that multiplies the
// transposed values into out (head columns x queries).  Queries stay in registers.
// The reference that the exponents are taken against follows the maximum only when
// that has grown by more than 2^8: sums stay far inside float and the rescaling of
// the output, 16 products per 32 columns, is rare.  Probabilities are rounded to the
// tensors' type for the second product (one rounding of each, of relative size
// 2^-9 in bf16); their sum is of the unrounded ones.
// A tile's keys and values go from memory to LDS without registers, one tile ahead.
// Bound: matrix instructions and LDS, each busy for 47% of the cycles (a wave reads a
// tile's 32 KB for 1,024 cycles of products), one after the other at two waves a SIMD.
// Measured: 2 x 8192 causal, 16 heads of 128, bf16: 561 us, 980 TFLOP/s (a large library
// product on the same card: 1,144).
template <class T, int DP>
__global__ __launch_bounds__(256, (kGroups<T, DP>)) void attention_forward_k(AttentionArgs a) {
    constexpr int N = kKeys<T>, kSub = N / 32, kBlocks = DP / 32, kSteps = DP / 16;
    using L = Tile<T, DP>;
    __shared__ __align__(16) char lds[2][2][N * L::kRowBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int pair = blockIdx.x % a.pairs, rest = blockIdx.x / a.pairs;
    // (long rows of a causal band first; a second round of workgroups comes to the CUs of
    // the first in the same order, so it goes the other way)
    const int split = rest / a.tiles, place = rest % a.tiles, tile = split & 1 ? place : a.tiles - 1 - place;
    const int b = pair / a.kv_heads, kv = pair % a.kv_heads;
    const Band band(a, b);
    const int rows = a.queries * a.group;
    const int row = tile * kBlockRows + wave * kWaveRows + (lane & 31);
    const int query = row / a.group, head = kv * a.group + row % a.group;
    const bool live = row < rows && query < band.ql;
    const int lo = live ? band.key_lo(query) : 0, hi = live ? band.key_hi(query) : 0;


    // the keys that the workgroup's rows, and this wave's, see at all, and those that
    // all of the wave's rows see
    const auto first_row = [&](int r) { return min(r / a.group, band.ql - 1); };
    const int block_first = tile * kBlockRows, wave_first = block_first + wave * kWaveRows;
    const bool any = block_first / a.group < band.ql, wave_any = wave_first / a.group < band.ql;
    int t0 = any ? band.key_lo(first_row(block_first)) / N : 0;
    int t1 = any ? (band.key_hi(first_row(block_first + kBlockRows - 1)) + N - 1) / N : 0;
    if (a.splits > 1) {
        const int share = (max(t1 - t0, 0) + a.splits - 1) / a.splits;
        t0 += split * share;
        t1 = min(t1, t0 + share);
    }
    const int wave_lo = wave_any ? band.key_lo(first_row(wave_first)) : 0;
    const int wave_hi = wave_any ? band.key_hi(first_row(wave_first + kWaveRows - 1)) : 0;
    const int full_lo = band.key_lo(first_row(wave_first + kWaveRows - 1));
    const int full_hi = wave_any && (wave_first + kWaveRows - 1) / a.group < band.ql ? band.key_hi(first_row(wave_first)) : 0;

    TileLoader<T, DP, N> kload, vload;
    kload.start(a.k.token, a.dim, a.wide_in);
    vload.start(a.v.token, a.dim, a.wide_in);
    const char* kbase = reinterpret_cast<const char*>(head_row<const T>(a.k, b, 0, kv));
    const char* vbase = reinterpret_cast<const char*>(head_row<const T>(a.v, b, 0, kv));
    const auto load = [&](int t, char* to_keys, char* to_values) __attribute__((always_inline)) {
        const int64_t first = int64_t(t) * N;
        kload.load(to_keys, kbase + first * kload.stride, band.kl - t * N, wave);
        vload.load(to_values, vbase + first * vload.stride, band.kl - t * N, wave);
    };

    Acc out[kBlocks] = {};
    float reference = -INFINITY, sum = 0;
    if (t0 < t1) {
        for (int i = 0; i < 4; ++i) kload.clear(lds[i >> 1][i & 1]);
        if (kload.direct && a.dim < DP) __syncthreads();
        load(t0, lds[0][0], lds[0][1]);
    }
    Frag<T> q[kSteps];
    load_fragments<T, DP>(q, head_row<const T>(a.q, b, query, head), a.dim, half, live, a.wide_in);
    // (the tile read and the tiles written do not overlap, which the compiler has to
    // know so as not to wait for the loads under way before it reads)
    const auto step = [&](int t, const char* __restrict__ keys, const char* __restrict__ values, char* __restrict__ next_keys,
                          char* __restrict__ next_values) __attribute__((always_inline)) {
        if (t + 1 < t1) load(t + 1, next_keys, next_values);
        const int first = t * N;
        if (first >= wave_hi || first + N <= wave_lo) return;
        Acc s[kSub];
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
            s[u] = Acc{};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) s[u] = mma(L::row(keys, 32 * u + (lane & 31), i, half), q[i], s[u]);
        }
        if (first < full_lo || first + N > full_hi) {
#pragma unroll
            for (int u = 0; u < kSub; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = first + 32 * u + 8 * (i >> 2) + 4 * half + (i & 3);
                    s[u][i] = key >= lo && key < hi ? s[u][i] : -INFINITY;
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
        top = halves_max(top) * a.scale2;
        const bool grown = top > reference + 8.f;
        if (__any(grown)) {
            const float next = grown ? top : reference, by = grown ? exp2_fast(reference - next) : 1.f;
            reference = next;
            sum *= by;
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) out[d] *= by;
        }
        const float base = reference == -INFINITY ? 0.f : reference;
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[u][i] = exp2_fast(fmaf(s[u][i], a.scale2, -base));
                sum += s[u][i];
            }
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const Frag<T> p = as_fragment<T>(s[u], i);
#pragma unroll
                for (int d = 0; d < kBlocks; ++d) out[d] = mma(L::column(values, d, 2 * u + i, lane), p, out[d]);
            }
    };
    for (int t = t0; t < t1; ++t) {
        const int now = (t - t0) & 1, next = now ^ 1;
        arrived();
        __syncthreads();
        step(t, lds[now][0], lds[now][1], lds[next][0], lds[next][1]);
    }
    sum = halves_sum(sum);
    if (row >= rows) return;
    if (a.splits > 1) {
        const int64_t at = (int64_t(split) * a.pairs + pair) * rows + row;
        if (half == 0) {
            a.part_stats[2 * at] = reference;
            a.part_stats[2 * at + 1] = sum;
        }
        if (sum != 0)
#pragma unroll
            for (int d = 0; d < kBlocks; ++d)
                store_column(a.part + at * a.dim, out[d], 1.f, d, half, a.dim, a.dim % 4 == 0);
        return;
    }
    if (sum == 0) clear(out);
    const float by = sum == 0 ? 0.f : 1.f / sum;
    T* to = head_row<T>(a.out, b, query, head);
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) store_column(to, out[d], by, d, half, a.dim, a.wide_out);
    if (a.lse && half == 0)
        a.lse[(int64_t(b) * a.kv_heads * a.group + head) * a.queries + query] =
            sum == 0 ? -INFINITY : reference * kLn2 + logf(sum);
}

// ---- one or two query rows: a vector kernel -------------------------------------------------
// One or two query rows of a key head read each key and value once, as they come
// from memory: LANES lanes hold a key's columns, eight each, and every row's query.
// Scores are summed over the lanes; each group of lanes keeps its own maximum and
// sum, joined at the end over the groups, the waves and (through memory, in
// attention_join_k) the splits.  Bound: HBM, and for short lists the latency of a
// launch and of a few rounds of loads, of which 16 waves need fewest.
template <int LANES>
__device__ inline float sum_lanes(float x) {
    // by cross-lane moves within rows of 16: neighbours, pairs, then mirror images
    const auto move = [](float v, auto control) {
        return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), decltype(control)::value, 0xf, 0xf, true));
    };
    x += move(x, std::integral_constant<int, 0xB1>{});                    // quad_perm [1,0,3,2]
    x += move(x, std::integral_constant<int, 0x4E>{});                    // quad_perm [2,3,0,1]
    if (LANES >= 8) x += move(x, std::integral_constant<int, 0x141>{});   // row_half_mirror
    if (LANES >= 16) x += move(x, std::integral_constant<int, 0x140>{});  // row_mirror
    return x;
}

template <class T>
__device__ inline void load8(float* v, const T* p, int left, bool wide) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int part = 0; part < 8; part += N) {
        if (wide) {
            vec<T, N> in = {};
            if (part < left) in = *reinterpret_cast<const vec<T, N>*>(p + part);
#pragma unroll
            for (int j = 0; j < N; ++j) v[part + j] = float(in[j]);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[part + j] = part + j < left ? float(p[part + j]) : 0.f;
        }
    }
}

constexpr int kStepDeep = 4;  // keys a group of lanes has under way
template <class T, int LANES, int R, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attention_step_k(AttentionArgs a) {
    constexpr int kGroupsOfWave = 64 / LANES, kAtOnce = WAVES * kGroupsOfWave, kDeep = kStepDeep;
    __shared__ float shared[WAVES][R][LANES * 8 + 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, in = lane % LANES, group = lane / LANES;
    const int pair = blockIdx.x % a.pairs, split = blockIdx.x / a.pairs;
    const int b = pair / a.kv_heads, kv = pair % a.kv_heads;
    const Band band(a, b);
    const int rows = a.queries * a.group, left = a.dim - in * 8;
    float q[R][8], acc[R][8] = {}, top[R], sum[R];
    int lo[R], hi[R], from = band.kl, to = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int query = r / a.group;
        const bool live = r < rows && query < band.ql;
        lo[r] = live ? band.key_lo(query) : 0;
        hi[r] = live ? band.key_hi(query) : 0;
        if (lo[r] < hi[r]) {
            from = min(from, lo[r]);
            to = max(to, hi[r]);
        }
        load8(q[r], head_row<const T>(a.q, b, query, kv * a.group + r % a.group) + in * 8, live ? left : 0, a.wide_in);
#pragma unroll
        for (int j = 0; j < 8; ++j) q[r][j] *= a.scale2;
        top[r] = -INFINITY;
        sum[r] = 0;
    }
    from = max(from, int(min(int64_t(split) * a.span, int64_t(band.kl))));
    to = int(min(int64_t(to), int64_t(split + 1) * a.span));
    const T* keys = head_row<const T>(a.k, b, 0, kv) + in * 8;
    const T* values = head_row<const T>(a.v, b, 0, kv) + in * 8;
    for (int first = from + wave * kGroupsOfWave + group; __any(first < to); first += kDeep * kAtOnce) {
        float k[kDeep][8], v[kDeep][8], s[kDeep][R];
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
            const int key = first + u * kAtOnce;
            load8(k[u], keys + int64_t(key) * a.k.token, key < to ? left : 0, a.wide_in);
        }
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
            const int key = first + u * kAtOnce;
            load8(v[u], values + int64_t(key) * a.v.token, key < to ? left : 0, a.wide_in);
        }
#pragma unroll
        for (int u = 0; u < kDeep; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float dot = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) dot = fmaf(q[r][j], k[u][j], dot);
                dot = sum_lanes<LANES>(dot);
                const int key = first + u * kAtOnce;
                s[u][r] = key >= lo[r] && key < hi[r] && key < to ? dot : -INFINITY;
            }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float next = top[r];
#pragma unroll
            for (int u = 0; u < kDeep; ++u) next = fmaxf(next, s[u][r]);
            const float base = next == -INFINITY ? 0.f : next, by = exp2_fast(top[r] - base);
            top[r] = next;
            sum[r] *= by;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[r][j] *= by;
#pragma unroll
            for (int u = 0; u < kDeep; ++u) {
                const float p = exp2_fast(s[u][r] - base);
                sum[r] += p;
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[r][j] = fmaf(p, v[u][j], acc[r][j]);
            }
        }
    }
    // the wave's groups, then the waves
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int d = LANES; d < 64; d <<= 1) {
            const float other = __shfl_xor(top[r], d), next = fmaxf(top[r], other);
            const float base = next == -INFINITY ? 0.f : next;
            const float mine = exp2_fast(top[r] - base), theirs = exp2_fast(other - base);
            top[r] = next;
            sum[r] = sum[r] * mine + __shfl_xor(sum[r], d) * theirs;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[r][j] = acc[r][j] * mine + __shfl_xor(acc[r][j], d) * theirs;
        }
        if (group == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) shared[wave][r][in * 8 + j] = acc[r][j];
            if (in == 0) {
                shared[wave][r][LANES * 8] = top[r];
                shared[wave][r][LANES * 8 + 1] = sum[r];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * LANES * 8; i += 64 * WAVES) {
        const int r = i / (LANES * 8), d = i % (LANES * 8);
        if (r >= rows || d >= a.dim) continue;
        float next = -INFINITY, total = 0, value = 0;
        for (int w = 0; w < WAVES; ++w) next = fmaxf(next, shared[w][r][LANES * 8]);
        const float base = next == -INFINITY ? 0.f : next;
        for (int w = 0; w < WAVES; ++w) {
            const float by = exp2_fast(shared[w][r][LANES * 8] - base);
            total += shared[w][r][LANES * 8 + 1] * by;
            value += shared[w][r][d] * by;
        }
        const int query = r / a.group, head = kv * a.group + r % a.group;
        if (a.splits > 1) {
            const int64_t at = (int64_t(split) * a.pairs + pair) * rows + r;
            a.part[at * a.dim + d] = value;
            if (d == 0) {
                a.part_stats[2 * at] = next;
                a.part_stats[2 * at + 1] = total;
            }
        } else {
            head_row<T>(a.out, b, query, head)[d] = T(total == 0 ? 0.f : value / total);
            if (a.lse && d == 0)
                a.lse[(int64_t(b) * a.kv_heads * a.group + head) * a.queries + query] =
                    total == 0 ? -INFINITY : next * kLn2 + logf(total);
        }
    }
}

// ---- 32 query rows a workgroup: matrix tiles on waves' own keys ------------------------------
// 32 query rows of a key head are one matrix tile's columns, so every wave of the
// workgroup holds them all and the waves share out the KEYS: each brings tiles of 32
// to its own part of LDS and computes on them in turn, with no barrier until their
// outputs are joined.  For one token, or a few, on long lists eight such waves a CU
// keep its share of memory busy (bound: HBM; 16 sequences of up to 32,768 keys, 4
// heads of 128, bf16: 537 MB in 109 us of this kernel, 4.9 TB/s); small sets get four times the
// workgroups of 128 rows, and waves that wait for different things (4 x 729 rows on
// 729 keys, 32 wide, f32: 20.6 us, 31 with 128 rows a workgroup; bound: the float
// instruction, 8.2 us, busy for 40% of the cycles, and the loads, which a wave waits for
// tile by tile).
template <class T, int DP>
constexpr int kRowWaves = DP * sizeof(T) <= 256 ? 4 : 2;
template <class T, int DP>
__global__ __launch_bounds__((64 * kRowWaves<T, DP>), 2) void attention_rows_k(AttentionArgs a) {
    constexpr int kWaves = kRowWaves<T, DP>, kBlocks = DP / 32, kSteps = DP / 16;
    constexpr int kHalf = 32 * DP * int(sizeof(T));  // bytes of a tile of keys
    constexpr int kPitch = DP + 4;                   // floats of a row of a wave's output in LDS
    using L = Tile<T, DP>;
    __shared__ __align__(16) char lds[kWaves][2 * kHalf > 32 * kPitch * 4 ? 2 * kHalf : 32 * kPitch * 4];
    __shared__ float joined[kWaves][2][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int pair = blockIdx.x % a.pairs, rest = blockIdx.x / a.pairs;
    const int first_row = (a.tiles - 1 - rest % a.tiles) * kWaveRows, split = rest / a.tiles;
    const int b = pair / a.kv_heads, kv = pair % a.kv_heads;
    const Band band(a, b);
    const int rows = a.queries * a.group, row = first_row + (lane & 31);
    const int query = row / a.group, head = kv * a.group + row % a.group;
    const bool live = row < rows && query < band.ql;
    const int lo = live ? band.key_lo(query) : 0, hi = live ? band.key_hi(query) : 0;
    // keys that any row, and that all rows, see (the rows that count are the first)
    const int top_query = first_row / a.group, last_query = (min(first_row + kWaveRows, rows) - 1) / a.group;
    const bool any = top_query < band.ql;
    const int last = min(last_query, band.ql - 1);
    const int from = any ? max(band.key_lo(top_query), int(min(int64_t(split) * a.span, int64_t(band.kl)))) : 0;
    const int to = any ? int(min(int64_t(band.key_hi(last)), int64_t(split + 1) * a.span)) : 0;
    // (rows past the length see none: a tile with such rows is never whole)
    const int full_lo = any ? band.key_lo(last) : 0, full_hi = any && last_query < band.ql ? band.key_hi(top_query) : 0;
    const int t0 = from / 32, t1 = from < to ? (to + 31) / 32 : t0;

    Frag<T> q[kSteps];
    load_fragments<T, DP>(q, head_row<const T>(a.q, b, query, head), a.dim, half, live, a.wide_in);
    WaveLoader<T, DP, 32> kload, vload;
    kload.start(a.k.token, a.dim, a.wide_in, lane);
    vload.start(a.v.token, a.dim, a.wide_in, lane);
    const char* kbase = reinterpret_cast<const char*>(head_row<const T>(a.k, b, 0, kv));
    const char* vbase = reinterpret_cast<const char*>(head_row<const T>(a.v, b, 0, kv));
    char* tile = lds[wave];
    const char* values = tile + kHalf;
    Acc out[kBlocks] = {};
    float reference = -INFINITY, sum = 0;
    kload.clear(tile, lane);
    vload.clear(tile + kHalf, lane);
    for (int t = t0 + wave; t < t1; t += kWaves) {
        kload.load(tile, kbase + int64_t(t) * 32 * kload.stride, band.kl - t * 32, lane);
        vload.load(tile + kHalf, vbase + int64_t(t) * 32 * vload.stride, band.kl - t * 32, lane);
        arrived();
        Acc s = {};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) s = mma(L::row(tile, lane & 31, i, half), q[i], s);
        const int first = t * 32;
        if (first < max(full_lo, from) || first + 32 > min(full_hi, to)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = first + 8 * (i >> 2) + 4 * half + (i & 3);
                s[i] = key >= max(lo, from) && key < min(hi, to) ? s[i] : -INFINITY;
            }
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        top = halves_max(top) * a.scale2;
        const bool grown = top > reference + 8.f;
        if (__any(grown)) {
            const float next = grown ? top : reference, by = grown ? exp2_fast(reference - next) : 1.f;
            reference = next;
            sum *= by;
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) out[d] *= by;
        }
        const float base = reference == -INFINITY ? 0.f : reference;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = exp2_fast(fmaf(s[i], a.scale2, -base));
            sum += s[i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const Frag<T> p = as_fragment<T>(s, i);
#pragma unroll
            for (int d = 0; d < kBlocks; ++d) out[d] = mma(L::column(values, d, i, lane), p, out[d]);
        }
    }
    sum = halves_sum(sum);
    // the waves' outputs side by side
    float* own = reinterpret_cast<float*>(tile);
    if (half == 0) {
        joined[wave][0][lane] = reference;
        joined[wave][1][lane] = sum;
    }
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) store_column(own + (lane & 31) * kPitch, out[d], 1.f, d, half, DP, true);
    __syncthreads();
    for (int i = threadIdx.x; i < min(kWaveRows, rows - first_row) * DP; i += 64 * kWaves) {
        const int r = i / DP, d = i % DP;
        if (d >= a.dim) continue;
        float next = -INFINITY, total = 0, value = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) next = fmaxf(next, joined[w][0][r]);
        const float base = next == -INFINITY ? 0.f : next;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float by = exp2_fast(joined[w][0][r] - base);
            total += joined[w][1][r] * by;
            value += reinterpret_cast<const float*>(lds[w])[r * kPitch + d] * by;
        }
        const int at_row = first_row + r, q = at_row / a.group, h = kv * a.group + at_row % a.group;
        if (a.splits > 1) {
            const int64_t at = (int64_t(split) * a.pairs + pair) * rows + at_row;
            a.part[at * a.dim + d] = value;
            if (d == 0) {
                a.part_stats[2 * at] = next;
                a.part_stats[2 * at + 1] = total;
            }
        } else {
            head_row<T>(a.out, b, q, h)[d] = T(total == 0 ? 0.f : value / total);
            if (a.lse && d == 0)
                a.lse[(int64_t(b) * a.kv_heads * a.group + h) * a.queries + q] =
                    total == 0 ? -INFINITY : next * kLn2 + logf(total);
        }
    }
}

// ---- joining splits -----------------------------------------------------------------------
struct Join {
    const float* part;
    HeadView out;
    int splits, rows, group, blocks;
    int teams;  // of 32 lanes a row, each with every teams-th split (a power of two)
    float scale;
};
struct JoinArgs {
    Join joins[3];
    const float* stats;  // null: plain sums
    float* lse;
    int pairs, dim, kv_heads, wide_part, wide_out;
};

// 32 lanes hold a row, four columns each; `teams` of them share its splits, with a
// running maximum each, and are joined through LDS in order.  Splits that saw no
// key wrote no output.  Bound: HBM (the parts read once; 64 splits of 256 rows of 128:
// 5.4 us).
template <class T>
__global__ __launch_bounds__(256) void attention_join_k(JoinArgs a) {
    int block = blockIdx.x, which = 0;
    while (block >= a.joins[which].blocks) block -= a.joins[which++].blocks;
    const Join c = a.joins[which];
    __shared__ float shared[8][32][6];
    const int lane = threadIdx.x & 31, team = threadIdx.x / 32, in = team & (c.teams - 1);
    const int64_t count = int64_t(a.pairs) * c.rows;
    const int64_t item = int64_t(block) * (8 / c.teams) + team / c.teams, at = min(item, count - 1);
    const int d = lane * 4;
    float top = -INFINITY, total = 0;
    vec<float, 4> value = {};
#pragma unroll 4
    for (int s = in; s < c.splits; s += c.teams) {
        const int64_t from = s * count + at;
        float m = 0, l = 1;
        if (a.stats) {
            const auto both = *reinterpret_cast<const vec<float, 2>*>(a.stats + 2 * from);
            m = both[0];
            l = both[1];
        }
        vec<float, 4> v = {};
        const float* p = c.part + from * a.dim + d;
        if (a.wide_part) {
            if (d < a.dim) v = *reinterpret_cast<const vec<float, 4>*>(p);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d + j < a.dim) v[j] = p[j];
        }
        if (a.stats) {
            const float next = fmaxf(top, m), base = next == -INFINITY ? 0.f : next;
            const float mine = exp2_fast(top - base), theirs = exp2_fast(m - base);
#pragma unroll
            for (int j = 0; j < 4; ++j) value[j] = value[j] * mine + (l == 0 ? 0.f : v[j] * theirs);
            total = total * mine + l * theirs;
            top = next;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) value[j] += v[j];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) shared[team][lane][j] = value[j];
    shared[team][lane][4] = top;
    shared[team][lane][5] = total;
    __syncthreads();
    if (in != 0 || item >= count) return;
    for (int t = 1; t < c.teams; ++t) {
        const float* other = shared[team + t][lane];
        if (a.stats) {
            const float next = fmaxf(top, other[4]), base = next == -INFINITY ? 0.f : next;
            const float mine = exp2_fast(top - base), theirs = exp2_fast(other[4] - base);
#pragma unroll
            for (int j = 0; j < 4; ++j) value[j] = value[j] * mine + other[j] * theirs;
            total = total * mine + other[5] * theirs;
            top = next;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) value[j] += other[j];
        }
    }
    const int pair = int(item / c.rows), row = int(item % c.rows);
    const int b = pair / a.kv_heads, kv = pair % a.kv_heads;
    const int token = row / c.group, head = kv * c.group + row % c.group;
    const float by = a.stats ? (total == 0 ? 0.f : 1.f / total) : c.scale;
    T* out = head_row<T>(c.out, b, token, head) + d;
    if (a.wide_out) {
        value *= by;
        if (d < a.dim) *reinterpret_cast<vec<T, 4>*>(out) = __builtin_convertvector(value, vec<T, 4>);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (d + j < a.dim) out[j] = T(value[j] * by);
    }
    if (a.lse && lane == 0)
        a.lse[(int64_t(b) * a.kv_heads * c.group + head) * (c.rows / c.group) + token] =
            total == 0 ? -INFINITY : top * kLn2 + logf(total);
}

// ---- gradient ---------------------------------------------------------------------------
// dout.out of every query row, and its lse in the scores' units (over the scale);
// sixteen lanes a row, rows from `first` on.  Bound: HBM (2 x 4096 x 16 rows of 128, bf16:
// 67 MB in 18 us).
template <class T>
__global__ __launch_bounds__(256) void attention_delta_k(AttentionArgs a, int64_t first) {
    const int heads = a.kv_heads * a.group;
    const int64_t count = int64_t(a.pairs / a.kv_heads) * a.queries * heads;
    const int64_t i = first + (blockIdx.x * 256u + threadIdx.x) / 16;
    const int in = threadIdx.x & 15;
    const int64_t item = min(i, count - 1);  // (all lanes take part in the sum)
    const int head = int(item % heads), query = int(item / heads % a.queries), b = int(item / heads / a.queries);
    const bool live = query < length_of(a.query_lengths, b, a.queries);
    float x[8], y[8], dot = 0;
    const int left = live ? a.dim - in * 8 : 0;
    load8(x, head_row<const T>(a.out, b, query, head) + in * 8, left, a.wide_in);
    load8(y, head_row<const T>(a.dout, b, query, head) + in * 8, left, a.wide_in);
#pragma unroll
    for (int j = 0; j < 8; ++j) dot = fmaf(x[j], y[j], dot);
    dot = sum_lanes<16>(dot);
    if (in == 0 && i < count) {
        const int64_t at = (int64_t(b) * heads + head) * a.queries + query;
        const float lse = live ? a.lse[at] : -INFINITY;
        // (no key: every probability is 0)
        a.row_lse[at] = lse == -INFINITY ? INFINITY : (lse - kLift<T> * kLn2) / a.scale;
        a.row_delta[at] = dot;
    }
}

// The statistics of a tile of queries, lse then delta, one a lane of one wave.
__device__ __attribute__((always_inline)) inline void load_statistics(const AttentionArgs& a, float* to, int64_t at, int valid,
                                                                      int lane) {
    const int i = fresh(lane);
    const float* from = (i < kQueries ? a.row_lse : a.row_delta) + at + min(i % kQueries, valid - 1);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 4, 0, 0);
}

// One tile of the gradients of a wave's 32 keys and values, which are in registers,
// over 32 queries: scores lie as queries x keys, so a lane holds 16 of the 32
// queries of ONE key, and its probabilities and score gradients are, in place, the
// fragments that multiply the transposed dout and queries into dv and dk.
template <class T, int DP>
__device__ __attribute__((always_inline)) inline void key_tile(const AttentionArgs& a, const Band& band, Fit<T>& fit,
                                                               Acc (&dk)[DP / 32], Acc* dv, const Frag<T>* k,
                                                               const Frag<T>* v, const char* queries,
                                                               const char* douts, const float* statistics, int first,
                                                               int key, bool hidden, int lane) {
    using L = Tile<T, DP>;
    const int now = fresh(lane), half = now >> 5;  // (addresses made anew: the gradients leave no registers for them)
    int lo = 0, hi = band.ql;
    if (hidden) {
        lo = key < band.kl ? band.query_lo(key) : 0;
        hi = key < band.kl ? band.query_hi(key) : 0;
    }
    // In 16 bits the products start from the rows' statistics (lse in the scores'
    // units), which so take no registers of their own; floats keep the bits that a
    // sum from a large start would round off.
    constexpr bool kFromStatistics = sizeof(T) == 2;
    Acc s = {}, dp = {}, lse, delta;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const auto l = *reinterpret_cast<const vec<float, 4>*>(statistics + 8 * g + 4 * half);
        const auto d = *reinterpret_cast<const vec<float, 4>*>(statistics + kQueries + 8 * g + 4 * half);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lse[4 * g + j] = -l[j];
            delta[4 * g + j] = -d[j];
        }
    }
    if constexpr (kFromStatistics) {
        s = lse;
        dp = delta;
    }
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) s = mma(L::row(queries, now & 31, i, half), k[i], s);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) dp = mma(L::row(douts, now & 31, i, half), v[i], dp);
    if constexpr (!kFromStatistics) {
        s += lse;
        dp += delta;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float p = exp2_fast(s[i] * a.scale2), ds = p * dp[i];
        if (hidden) {
            const int query = first + 8 * (i >> 2) + 4 * half + (i & 3);
            const bool seen = query >= lo && query < hi;
            p = seen ? p : 0.f;
            ds = seen ? ds : 0.f;
        }
        s[i] = p;
        dp[i] = ds;
    }
    fit(dp, dk);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const Frag<T> p = as_fragment<T>(s, i), ds = as_fragment<T>(dp, i);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
            dv[d] = mma(L::column(douts, d, i, now), p, dv[d]);
            dk[d] = mma(L::column(queries, d, i, now), ds, dk[d]);
        }
    }
}

// One tile of 32 keys of the gradient of a wave's 32 query rows: the forward's
// shape, with queries and dout in registers.
template <class T, int DP>
__device__ __attribute__((always_inline)) inline void query_tile(const AttentionArgs& a, Fit<T>& fit, Acc (&dq)[DP / 32],
                                                                 const Frag<T>* q,
                                                                 const Frag<T>* dout, const char* keys,
                                                                 const char* values, int at, int first, int lo, int hi,
                                                                 bool hidden, float lse, float delta, int lane) {
    using L = Tile<T, DP>;
    const int half = lane >> 5;
    Acc s = {}, dp = {};
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) s = mma(L::row(keys, at + (lane & 31), i, half), q[i], s);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) dp = mma(L::row(values, at + (lane & 31), i, half), dout[i], dp);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int key = first + 8 * (i >> 2) + 4 * half + (i & 3);
        float ds = exp2_fast((s[i] - lse) * a.scale2) * (dp[i] - delta);
        if (hidden) ds = key >= lo && key < hi ? ds : 0.f;
        s[i] = ds;
    }
    fit(s, dq);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const Frag<T> ds = as_fragment<T>(s, i);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) dq[d] = mma(L::column(keys, d, at / 16 + i, lane), ds, dq[d]);
    }
}

// A wave's gradient columns (32 rows of DP) times `by` into its place in LDS, and the four
// waves' sums of it by all of them: column(row, d, value).
template <int DP>
constexpr int kPitch = DP + 4;  // floats of a row there
template <int DP, class F>
__device__ inline void join_waves(float* const (&places)[4], const Acc* c, float by, int wave, int lane, int rows, int dim,
                                  F column) {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) store_column(places[wave] + (lane & 31) * kPitch<DP>, c[d], by, d, lane >> 5, DP, true);
    __syncthreads();
    for (int i = threadIdx.x; i < rows * DP; i += 256) {
        const int row = i / DP, d = i % DP, at = row * kPitch<DP> + d;
        if (d < dim) column(row, d, (places[0][at] + places[1][at]) + (places[2][at] + places[3][at]));
    }
    __syncthreads();
}

// Gradients of keys and values.  128 keys a workgroup, 32 a wave, over tiles of 32
// queries of every head that reads them, one ahead in LDS of the one computed on.
template <class T, int DP>
struct KeyShared {
    char tiles[2][2][kQueries * Tile<T, DP>::kRowBytes];
    float stats[2][2][kQueries];
};
template <class T, int DP>
__device__ __attribute__((always_inline)) inline void key_gradient(const AttentionArgs& a, int block, KeyShared<T, DP>& shared) {
    constexpr int kBlocks = DP / 32, kSteps = DP / 16;
    auto& lds = shared.tiles;
    auto& stats = shared.stats;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int pair = block % a.pairs, rest = block / a.pairs;
    // (a causal band's first keys are seen most; a second round of workgroups comes to
    // the CUs of the first in the same order, so it goes the other way)
    const int split = rest / a.key_tiles, place = rest % a.key_tiles, tile = split & 1 ? a.key_tiles - 1 - place : place;
    const int b = pair / a.kv_heads, kv = pair % a.kv_heads;
    const Band band(a, b);
    const int block_first = tile * kBlockRows, wave_first = block_first + wave * kWaveRows;
    const int key = wave_first + (lane & 31);
    const bool live = key < band.kl;

    const auto last = [&](int j) { return min(j, band.kl - 1); };
    const bool any = block_first < band.kl, wave_any = wave_first < band.kl;
    const int t0 = any ? band.query_lo(block_first) / kQueries : 0;
    const int t1 = any ? (band.query_hi(last(block_first + kBlockRows - 1)) + kQueries - 1) / kQueries : 0;
    const int per_head = max(t1 - t0, 0);
    int from = 0, to = per_head * a.group;
    if (a.key_splits > 1) {
        const int share = (to + a.key_splits - 1) / a.key_splits;
        from = min(split * share, to);
        to = min(to, from + share);
    }
    const int wave_lo = wave_any ? band.query_lo(wave_first) : 0;
    const int wave_hi = wave_any ? band.query_hi(last(wave_first + kWaveRows - 1)) : 0;
    const int full_lo = band.query_lo(last(wave_first + kWaveRows - 1));
    const int full_hi = wave_first + kWaveRows <= band.kl ? band.query_hi(wave_first) : 0;

    TileLoader<T, DP, kQueries> qload, oload;
    qload.start(a.q.token, a.dim, a.wide_in);
    oload.start(a.dout.token, a.dim, a.wide_in);
    // the next load: tile t of a head, and where it lies; after a head's last tile the
    // next head's first
    const int head = per_head ? from / per_head : 0;
    int t = t0 + from - head * per_head;
    const int first_head = kv * a.group + head;
    const char* at_q = reinterpret_cast<const char*>(head_row<const T>(a.q, b, int64_t(t) * kQueries, first_head));
    const char* at_o = reinterpret_cast<const char*>(head_row<const T>(a.dout, b, int64_t(t) * kQueries, first_head));
    int64_t at_s = (int64_t(b) * a.kv_heads * a.group + first_head) * a.queries + int64_t(t) * kQueries;
    const int64_t back_q = a.q.head * int64_t(sizeof(T)) - int64_t(per_head) * kQueries * qload.stride;
    const int64_t back_o = a.dout.head * int64_t(sizeof(T)) - int64_t(per_head) * kQueries * oload.stride;
    const auto load = [&](char* to_queries, char* to_douts, float* to_stats) __attribute__((always_inline)) {
        const int valid = band.ql - t * kQueries;
        qload.load(to_queries, at_q, valid, wave);
        oload.load(to_douts, at_o, valid, wave);
        if (wave == 0) load_statistics(a, to_stats, at_s, valid, lane);
        at_q += kQueries * qload.stride;
        at_o += kQueries * oload.stride;
        at_s += kQueries;
        if (++t == t1) {
            t = t0;
            at_q += back_q;
            at_o += back_o;
            at_s += a.queries - per_head * kQueries;
        }
    };

    Acc dk[kBlocks] = {}, dv[kBlocks] = {};
    Fit<T> fit;
    if (from < to) {
        for (int i = 0; i < 4; ++i) qload.clear(lds[i >> 1][i & 1]);
        if (qload.direct && a.dim < DP) __syncthreads();
    }
    int at = t;  // of the tile computed on
    if (from < to) load(lds[0][0], lds[0][1], stats[0][0]);
    Frag<T> k[kSteps], v[kSteps];
    load_fragments<T, DP>(k, head_row<const T>(a.k, b, key, kv), a.dim, half, live, a.wide_in);
    load_fragments<T, DP>(v, head_row<const T>(a.v, b, key, kv), a.dim, half, live, a.wide_in);
    const auto step = [&](bool more, const char* __restrict__ queries, const char* __restrict__ douts,
                          const float* __restrict__ statistics, char* __restrict__ next_queries,
                          char* __restrict__ next_douts, float* __restrict__ next_statistics) __attribute__((always_inline)) {
        const int first = at * kQueries;
        if (++at == t1) at = t0;
        if (more) load(next_queries, next_douts, next_statistics);
        if (first >= wave_hi || first + kQueries <= wave_lo) return;
        key_tile<T, DP>(a, band, fit, dk, dv, k, v, queries, douts, statistics, first, key,
                        first < full_lo || first + kQueries > full_hi, lane);
    };
    for (int i = from; i < to; ++i) {
        const int now = (i - from) & 1, next = now ^ 1;
        arrived();
        __syncthreads();
        step(i + 1 < to, lds[now][0], lds[now][1], stats[now][0], lds[next][0], lds[next][1], stats[next][0]);
    }
    const int end = fresh(lane), last_key = wave_first + (end & 31), last_half = end >> 5;
    if (last_key >= a.keys) return;
    const float off = fit.off();
    if (!seen(band, last_key)) {
        clear(dk);
        clear(dv);
    }
    if (a.key_splits > 1) {
        // [which][split][pair][key][dim]
        const int64_t at = (int64_t(split) * a.pairs + pair) * a.keys + last_key;
        const int64_t other = int64_t(a.key_splits) * a.pairs * a.keys;
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) {
            store_column(a.key_part + at * a.dim, dk[d], off, d, last_half, a.dim, a.dim % 4 == 0);
            store_column(a.key_part + (other + at) * a.dim, dv[d], fit.p_off(), d, last_half, a.dim, a.dim % 4 == 0);
        }
        return;
    }
    T *to_k = head_row<T>(a.dk, b, last_key, kv), *to_v = head_row<T>(a.dv, b, last_key, kv);
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) {
        store_column(to_k, dk[d], off * a.scale, d, last_half, a.dim, a.wide_out);
        store_column(to_v, dv[d], fit.p_off(), d, last_half, a.dim, a.wide_out);
    }
}

// Gradients of queries, 128 rows a workgroup.  (A second pass over the scores, so
// that no two workgroups add to one place: two products of nine, for sums in a fixed
// order and no float copy of dq.)
template <class T, int DP>
struct QueryShared {
    char tiles[2][2][kKeys<T> * Tile<T, DP>::kRowBytes];
};
template <class T, int DP>
__device__ __attribute__((always_inline)) inline void query_gradient(const AttentionArgs& a, int block, QueryShared<T, DP>& shared) {
    constexpr int N = kKeys<T>, kBlocks = DP / 32, kSteps = DP / 16;
    auto& lds = shared.tiles;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int pair = block % a.pairs, rest = block / a.pairs;
    const int split = rest / a.tiles, place = rest % a.tiles, tile = split & 1 ? place : a.tiles - 1 - place;
    const int b = pair / a.kv_heads, kv = pair % a.kv_heads;
    const Band band(a, b);
    const int rows = a.queries * a.group;
    const int row = tile * kBlockRows + wave * kWaveRows + (lane & 31);
    const int query = row / a.group, head = kv * a.group + row % a.group;
    const bool live = row < rows && query < band.ql;
    const int lo = live ? band.key_lo(query) : 0, hi = live ? band.key_hi(query) : 0;

    const auto first_row = [&](int r) { return min(r / a.group, band.ql - 1); };
    const int block_first = tile * kBlockRows, wave_first = block_first + wave * kWaveRows;
    const bool any = block_first / a.group < band.ql, wave_any = wave_first / a.group < band.ql;
    int t0 = any ? band.key_lo(first_row(block_first)) / N : 0;
    int t1 = any ? (band.key_hi(first_row(block_first + kBlockRows - 1)) + N - 1) / N : 0;
    if (a.splits > 1) {
        const int share = (max(t1 - t0, 0) + a.splits - 1) / a.splits;
        t0 += split * share;
        t1 = min(t1, t0 + share);
    }
    const int wave_lo = wave_any ? band.key_lo(first_row(wave_first)) : 0;
    const int wave_hi = wave_any ? band.key_hi(first_row(wave_first + kWaveRows - 1)) : 0;
    const int full_lo = band.key_lo(first_row(wave_first + kWaveRows - 1));
    const int full_hi = wave_any && (wave_first + kWaveRows - 1) / a.group < band.ql ? band.key_hi(first_row(wave_first)) : 0;

    TileLoader<T, DP, N> kload, vload;
    kload.start(a.k.token, a.dim, a.wide_in);
    vload.start(a.v.token, a.dim, a.wide_in);
    const char* kbase = reinterpret_cast<const char*>(head_row<const T>(a.k, b, 0, kv));
    const char* vbase = reinterpret_cast<const char*>(head_row<const T>(a.v, b, 0, kv));
    const auto load = [&](int t, char* to_keys, char* to_values) __attribute__((always_inline)) {
        const int64_t first = int64_t(t) * N;
        kload.load(to_keys, kbase + first * kload.stride, band.kl - t * N, wave);
        vload.load(to_values, vbase + first * vload.stride, band.kl - t * N, wave);
    };

    Acc dq[kBlocks] = {};
    Fit<T> fit;
    if (t0 < t1) {
        for (int i = 0; i < 4; ++i) kload.clear(lds[i >> 1][i & 1]);
        if (kload.direct && a.dim < DP) __syncthreads();
        load(t0, lds[0][0], lds[0][1]);
    }
    Frag<T> q[kSteps], dout[kSteps];
    load_fragments<T, DP>(q, head_row<const T>(a.q, b, query, head), a.dim, half, live, a.wide_in);
    load_fragments<T, DP>(dout, head_row<const T>(a.dout, b, query, head), a.dim, half, live, a.wide_in);
    const int64_t at_row = (int64_t(b) * a.kv_heads * a.group + head) * a.queries + query;
    const float lse = live ? a.row_lse[at_row] : INFINITY, delta = live ? a.row_delta[at_row] : 0.f;
    const auto step = [&](int t, const char* __restrict__ keys, const char* __restrict__ values, char* __restrict__ next_keys,
                          char* __restrict__ next_values) __attribute__((always_inline)) {
        if (t + 1 < t1) load(t + 1, next_keys, next_values);
        const int first = t * N;
        if (first >= wave_hi || first + N <= wave_lo) return;
        const bool hidden = first < full_lo || first + N > full_hi;
#pragma unroll
        for (int u = 0; u < N; u += 32)
            query_tile<T, DP>(a, fit, dq, q, dout, keys, values, u, first + u, lo, hi, hidden, lse, delta, lane);
    };
    for (int t = t0; t < t1; ++t) {
        const int now = (t - t0) & 1, next = now ^ 1;
        arrived();
        __syncthreads();
        step(t, lds[now][0], lds[now][1], lds[next][0], lds[next][1]);
    }
    if (row >= rows) return;
    if (lo >= hi) clear(dq);
    const float off = fit.off();
    if (a.splits > 1) {
        const int64_t at = (int64_t(split) * a.pairs + pair) * rows + row;
#pragma unroll
        for (int d = 0; d < kBlocks; ++d)
            store_column(a.part + at * a.dim, dq[d], off, d, half, a.dim, a.dim % 4 == 0);
        return;
    }
    T* to = head_row<T>(a.dq, b, query, head);
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) store_column(to, dq[d], off * a.scale, d, half, a.dim, a.wide_out);
}

// Both in one launch, the keys' workgroups first (four products to three): where
// either would leave the device short of workgroups the other fills it.  Score
// gradients are rounded to the tensors' type for the products that sum them.  Bound:
// as the forward's (busy 40% and 43%); at 128 columns of 16 bits a wave's keys, values and
// their gradients leave 32 of its 256 registers.  Measured: 2 x 4096 causal, 16 heads on
// 4, 128 wide, bf16: 531 us for seven products, 906 TFLOP/s.
template <class T, int DP>
__global__ __launch_bounds__(256, (kGroups<T, DP>)) void attention_gradient_k(AttentionArgs a) {
    __shared__ __align__(16) union {
        KeyShared<T, DP> key;
        QueryShared<T, DP> query;
    } shared;
    if (int(blockIdx.x) < a.key_blocks) key_gradient<T, DP>(a, blockIdx.x, shared.key);
    else query_gradient<T, DP>(a, blockIdx.x - a.key_blocks, shared.query);
}

// The same for small sets, 32 keys or rows a workgroup, whose waves share out the
// tiles of the other axis, each in its own part of LDS, and are joined at the end:
// four times the workgroups, nothing to join in memory.  (8 x 729 points, 4 heads of
// 32, f32: 88 us with the launch before it, 107 with 128 a workgroup; bound: the
// float instruction, 50 us for seven products.)
template <class T, int DP>
struct FewShared {
    static constexpr int kTiles = 2 * 32 * Tile<T, DP>::kRowBytes, kOut = 32 * kPitch<DP> * 4;
    char tiles[4][kTiles > kOut ? kTiles : kOut];
    float stats[4][2][kQueries];
};
template <class T, int DP>
__device__ __attribute__((always_inline)) inline void few_keys_gradient(const AttentionArgs& a, int block, FewShared<T, DP>& shared) {
    constexpr int kBlocks = DP / 32, kSteps = DP / 16, kHalf = 32 * Tile<T, DP>::kRowBytes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int pair = block % a.pairs, first_key = block / a.pairs * kWaveRows;
    const int b = pair / a.kv_heads, kv = pair % a.kv_heads;
    const Band band(a, b);
    const int key = first_key + (lane & 31), last = min(first_key + kWaveRows, band.kl) - 1;
    const bool any = first_key < band.kl, live = key < band.kl;
    const int lo = any ? band.query_lo(first_key) : 0, hi = any ? band.query_hi(last) : 0;
    const int full_lo = any ? band.query_lo(last) : 0;
    const int full_hi = first_key + kWaveRows <= band.kl ? band.query_hi(first_key) : 0;
    const int t0 = lo / kQueries, per_head = lo < hi ? (hi + kQueries - 1) / kQueries - t0 : 0;

    Frag<T> k[kSteps], v[kSteps];
    load_fragments<T, DP>(k, head_row<const T>(a.k, b, key, kv), a.dim, half, live, a.wide_in);
    load_fragments<T, DP>(v, head_row<const T>(a.v, b, key, kv), a.dim, half, live, a.wide_in);
    WaveLoader<T, DP, 32> qload, oload;
    qload.start(a.q.token, a.dim, a.wide_in, lane);
    oload.start(a.dout.token, a.dim, a.wide_in, lane);
    char* tile = shared.tiles[wave];
    float* stats = shared.stats[wave][0];
    qload.clear(tile, lane);
    oload.clear(tile + kHalf, lane);
    Acc dk[kBlocks] = {}, dv[kBlocks] = {};
    Fit<T> fit;
    for (int i = wave; i < per_head * a.group; i += 4) {
        const int head = kv * a.group + i / per_head, first = (t0 + i % per_head) * kQueries, valid = band.ql - first;
        qload.load(tile, reinterpret_cast<const char*>(head_row<const T>(a.q, b, first, head)), valid, lane);
        oload.load(tile + kHalf, reinterpret_cast<const char*>(head_row<const T>(a.dout, b, first, head)), valid, lane);
        load_statistics(a, stats, (int64_t(b) * a.kv_heads * a.group + head) * a.queries + first, valid, lane);
        arrived();
        key_tile<T, DP>(a, band, fit, dk, dv, k, v, tile, tile + kHalf, stats, first, key,
                        first < full_lo || first + kQueries > full_hi, lane);
    }
    float* const places[4] = {reinterpret_cast<float*>(shared.tiles[0]), reinterpret_cast<float*>(shared.tiles[1]),
                              reinterpret_cast<float*>(shared.tiles[2]), reinterpret_cast<float*>(shared.tiles[3])};
    if (!seen(band, key)) {
        clear(dk);
        clear(dv);
    }
    const int rows = min(kWaveRows, a.keys - first_key);
    join_waves<DP>(places, dk, fit.off(), wave, lane, rows, a.dim, [&](int r, int d, float x) {
        head_row<T>(a.dk, b, first_key + r, kv)[d] = T(x * a.scale);
    });
    join_waves<DP>(places, dv, fit.p_off(), wave, lane, rows, a.dim, [&](int r, int d, float x) {
        head_row<T>(a.dv, b, first_key + r, kv)[d] = T(x);
    });
}
template <class T, int DP>
__device__ __attribute__((always_inline)) inline void few_rows_gradient(const AttentionArgs& a, int block, FewShared<T, DP>& shared) {
    constexpr int kBlocks = DP / 32, kSteps = DP / 16, kHalf = 32 * Tile<T, DP>::kRowBytes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int pair = block % a.pairs, first_row = (a.tiles - 1 - block / a.pairs) * kWaveRows;
    const int b = pair / a.kv_heads, kv = pair % a.kv_heads;
    const Band band(a, b);
    const int rows = a.queries * a.group, row = first_row + (lane & 31);
    const int query = row / a.group, head = kv * a.group + row % a.group;
    const bool live = row < rows && query < band.ql;
    const int lo = live ? band.key_lo(query) : 0, hi = live ? band.key_hi(query) : 0;
    const int top_query = first_row / a.group, last_query = (min(first_row + kWaveRows, rows) - 1) / a.group;
    const bool any = top_query < band.ql;
    const int last = min(last_query, band.ql - 1);
    const int from = any ? band.key_lo(top_query) : 0, to = any ? band.key_hi(last) : 0;
    const int full_lo = any ? band.key_lo(last) : 0, full_hi = any && last_query < band.ql ? band.key_hi(top_query) : 0;

    Frag<T> q[kSteps], dout[kSteps];
    load_fragments<T, DP>(q, head_row<const T>(a.q, b, query, head), a.dim, half, live, a.wide_in);
    load_fragments<T, DP>(dout, head_row<const T>(a.dout, b, query, head), a.dim, half, live, a.wide_in);
    const int64_t at_row = (int64_t(b) * a.kv_heads * a.group + head) * a.queries + query;
    const float lse = live ? a.row_lse[at_row] : INFINITY, delta = live ? a.row_delta[at_row] : 0.f;
    WaveLoader<T, DP, 32> kload, vload;
    kload.start(a.k.token, a.dim, a.wide_in, lane);
    vload.start(a.v.token, a.dim, a.wide_in, lane);
    const char* kbase = reinterpret_cast<const char*>(head_row<const T>(a.k, b, 0, kv));
    const char* vbase = reinterpret_cast<const char*>(head_row<const T>(a.v, b, 0, kv));
    char* tile = shared.tiles[wave];
    kload.clear(tile, lane);
    vload.clear(tile + kHalf, lane);
    Acc dq[kBlocks] = {};
    Fit<T> fit;
    for (int t = from / 32 + wave; t * 32 < to; t += 4) {
        const int first = t * 32;
        kload.load(tile, kbase + int64_t(first) * kload.stride, band.kl - first, lane);
        vload.load(tile + kHalf, vbase + int64_t(first) * vload.stride, band.kl - first, lane);
        arrived();
        query_tile<T, DP>(a, fit, dq, q, dout, tile, tile + kHalf, 0, first, lo, hi, first < full_lo || first + 32 > full_hi, lse,
                          delta, lane);
    }
    if (lo >= hi) clear(dq);
    float* const places[4] = {reinterpret_cast<float*>(shared.tiles[0]), reinterpret_cast<float*>(shared.tiles[1]),
                              reinterpret_cast<float*>(shared.tiles[2]), reinterpret_cast<float*>(shared.tiles[3])};
    join_waves<DP>(places, dq, fit.off(), wave, lane, min(kWaveRows, rows - first_row), a.dim, [&](int r, int d, float x) {
        const int at = first_row + r;
        head_row<T>(a.dq, b, at / a.group, kv * a.group + at % a.group)[d] = T(x * a.scale);
    });
}
template <class T, int DP>
__global__ __launch_bounds__(256, (kGroups<T, DP>)) void attention_few_gradient_k(AttentionArgs a) {
    __shared__ __align__(16) FewShared<T, DP> shared;
    if (int(blockIdx.x) < a.key_blocks) few_keys_gradient<T, DP>(a, blockIdx.x, shared);
    else few_rows_gradient<T, DP>(a, blockIdx.x - a.key_blocks, shared);
}

// ---- host -----------------------------------------------------------------------------------
int ceil_div(int64_t a, int64_t b) { return int((a + b - 1) / b); }

int step_lanes(int dim) { return dim <= 32 ? 4 : dim <= 64 ? 8 : 16; }

// What a launch of `blocks` workgroups in `splits` each takes, in us: the longest
// workgroup on a CU of its own, or all of them on the CUs they share, with their
// starts; then the join, whose parts are written and read once.  Its constants were set
// on calls of 729 to 8192 rows and keys.
struct Work {
    int64_t blocks = 0;               // before splitting
    double longest = 0, mean = 0;     // steps of 32 keys (or queries) of a workgroup
    double alone = 0, shared = 0;     // us a step, on a CU of its own and in its share of a full one
    double part_bytes = 0;            // a split writes
};
double launch_time(const Work* w, const int* splits, int count, int cus) {
    double longest = 0, all = 0, blocks = 0, join = 0;
    for (int i = 0; i < count; ++i) {
        longest = std::max(longest, w[i].longest / splits[i] * w[i].alone);
        all += w[i].blocks * w[i].mean * w[i].shared / cus;
        blocks += double(w[i].blocks) * splits[i];
        if (splits[i] > 1) join = std::max(join, 6.0) + w[i].part_bytes * splits[i] / 1e6;
    }
    const double rounds = std::ceil(blocks / cus);
    if (blocks > 0) all *= rounds * cus / blocks;  // (the last round leaves CUs idle)
    return std::max(longest, all) + 2.5 * rounds + join;
}

// How the launches of a shape are cut, the same for every call: work is split over
// the long axis and joined where whole rows would leave the device short of
// workgroups.
void cut_launches(Attention& p) {
    const auto& s = p.shape;
    Cut& c = p.cut;
    const int64_t group = s.heads / s.kv_heads, pairs = int64_t(s.batch) * s.kv_heads;
    c.rows = int(s.query_tokens * group);
    c.row_tiles = ceil_div(c.rows, kBlockRows);
    c.key_tiles = ceil_div(s.key_tokens, kBlockRows);
    const int cus = p.dev->compute_units;
    const bool floats = s.dtype == CPDE_F32;
    // us of a step of two products (32 queries of every wave on 32 keys)
    const double alone = floats ? 0.35 + 0.0344 * s.head_dim : 0.4 + 0.004 * s.head_dim;
    const double shared = floats ? 0.0355 * s.head_dim : 0.15 + 0.0037 * s.head_dim;
    // a band bounded on one side shows half of the other axis on average, on both sides its width
    const auto seen = [&](double steps) {
        const double width = s.left >= 0 && s.right >= 0 ? (double(s.left) + s.right + kBlockRows) / 32 : 2 * steps;
        return std::min({steps, width, s.left >= 0 || s.right >= 0 ? std::max(steps / 2, 1.0) : steps});
    };
    const double key_steps = ceil_div(s.key_tokens, 32), query_steps = ceil_div(s.query_tokens, 32);
    const Work rows{pairs * c.row_tiles, s.left >= 0 && s.right >= 0 ? seen(key_steps) : key_steps, seen(key_steps), alone,
                    shared, 4.0 * double(pairs) * c.rows * s.head_dim};
    constexpr int kMostSplits = 64;
    // The vector kernel takes one or two rows of floats, or of a list short enough for
    // one workgroup's few rounds; matrix tiles the others (us, vector and tiles; 8 x 8192
    // keys of 4 heads: f32, 128 wide, 1 row 61 and 75, 4 rows 75 and 77; bf16, 1 row 50
    // and 32, 2 rows 55 and 32; 729 keys of 4 heads: bf16, 128 wide, 1 row 8.6 and 11.2).
    const int round = kStepDeep * 16 * (64 / step_lanes(s.head_dim));
    c.brief = s.key_tokens <= 2 * round;
    c.step = c.rows <= kStepRows && (c.brief || floats);
    if (c.step) {
        // 16 workgroups of four waves a CU, in whole rounds of a workgroup's loads; a
        // short list in one of 16 waves
        const int64_t share = c.brief ? s.key_tokens : ceil_div(pairs * s.key_tokens, 16 * cus);
        c.span = std::max(ceil_div(std::max<int64_t>(share, 1), round / 4) * (round / 4), round / 4);
        c.forward = std::max(ceil_div(s.key_tokens, c.span), 1);
    } else {
        double best = 0;
        for (int n = 1; n <= std::clamp<int>(int(key_steps) / 4, 1, kMostSplits); ++n) {
            const double time = launch_time(&rows, &n, 1, cus);
            if (n == 1 || time < best) best = time, c.forward = n;
        }
        // 32 rows a workgroup, its waves sharing the keys: the steps of 128 rows' workgroups
        // over waves, each a little dearer, as many of them, and waves to join
        const int tiles = 32 * (s.head_dim * type_bytes(s.dtype) <= 256 ? 4 : 2), waves = tiles / 32;
        const double blocks = double(pairs) * ceil_div(c.rows, kWaveRows), steps = std::ceil(key_steps / waves);
        const double dearer = floats ? 1.2 : 1.45, fixed = 3.5 + 1.5 * std::ceil(blocks / cus);
        const double few = std::max(steps * alone, blocks * std::ceil(seen(key_steps) / waves) * waves / 4 * dearer * shared / cus) + fixed;
        if (c.rows <= kWaveRows) {
            // memory's time, not a wave's: eight workgroups a CU, of at least four tiles a wave
            c.few = true;
            const int64_t share = std::max<int64_t>(ceil_div(pairs * s.key_tokens, 8 * cus), 4 * tiles);
            c.span = ceil_div(share, tiles) * tiles;
            c.forward = std::max(ceil_div(s.key_tokens, c.span), 1);
        } else if (few < best) {
            c.few = true;
            c.span = std::max(ceil_div(s.key_tokens, tiles), 1) * tiles;
            c.forward = 1;
        }
    }
    size_t part = 0;
    if (c.forward > 1) {
        part = size_t(c.forward) * pairs * c.rows * s.head_dim;
        c.part_stats = size_t(c.forward) * pairs * c.rows * 2;
    }
    if (s.backward) {
        const double per_head = s.left >= 0 && s.right >= 0 ? seen(query_steps) : query_steps;
        const Work both[2] = {{pairs * c.key_tiles, group * per_head, group * seen(query_steps), 2 * alone, 2 * shared,
                               8.0 * double(pairs) * s.key_tokens * s.head_dim},
                              {rows.blocks, rows.longest, rows.mean, 1.5 * alone, 1.5 * shared, rows.part_bytes}};
        double best = 0;
        const int most_keys = std::clamp<int>(int(std::min(group * query_steps, 1e6)) / 4, 1, kMostSplits);
        const int most_queries = std::clamp<int>(int(key_steps) / 4, 1, kMostSplits);
        for (int k = 1; k <= most_keys; ++k)
            for (int q = 1; q <= most_queries; ++q) {
                const int n[2] = {k, q};
                const double time = launch_time(both, n, 2, cus);
                if ((k == 1 && q == 1) || time < best) best = time, c.key = k, c.query = q;
            }
        // 32 keys or rows a workgroup, as above; two outputs to join
        const double blocks[2] = {double(pairs) * ceil_div(s.key_tokens, kWaveRows), double(pairs) * ceil_div(c.rows, kWaveRows)};
        const double few = std::max({std::ceil(both[0].longest / 4) * both[0].alone, std::ceil(both[1].longest / 4) * both[1].alone,
                                     (blocks[0] * std::ceil(both[0].mean / 4) * both[0].shared +
                                      blocks[1] * std::ceil(both[1].mean / 4) * both[1].shared) * (floats ? 1.1 : 1.45) / cus}) +
                           3.5 + 2 * std::ceil((blocks[0] + blocks[1]) / cus);
        c.few_gradient = few < best;
        if (c.few_gradient) c.key = c.query = 1;
        if (c.query > 1) part = std::max(part, size_t(c.query) * pairs * c.rows * s.head_dim);
        if (c.key > 1) c.key_part = 2 * size_t(c.key) * pairs * s.key_tokens * s.head_dim;
        c.stats = 2 * size_t(s.batch) * s.heads * s.query_tokens;
    }
    const auto padded = [](size_t n) { return (n + 63) / 64 * 64; };
    c.stats = padded(c.stats);
    c.part = padded(part);
    c.part_stats = padded(c.part_stats);
    c.floats = c.stats + c.part + c.part_stats + c.key_part;
}

// Pairs of a query and a key that it sees, at the full lengths.
double seen_pairs(const cpde_attention_shape& s) {
    const int64_t n = s.query_tokens, m = s.key_tokens;
    // x clamped to 0..m, summed over n values from `first` on
    const auto clamped = [&](int64_t first) {
        const auto below = [&](int64_t end) {
            const int64_t ramp = std::clamp<int64_t>(end, 0, m);
            return double(ramp) * double(ramp - 1) / 2 + double(std::max<int64_t>(end, 0) - ramp) * double(m);
        };
        return below(first + n) - below(first);
    };
    return (s.right < 0 ? double(n) * double(m) : clamped(m - n + s.right + 1)) - (s.left < 0 ? 0 : clamped(m - n - s.left));
}

HeadView view(const cpde_heads& h) { return {static_cast<char*>(h.data), h.batch, h.token, h.head}; }

// Checks a tensor's address and strides; returns whether it takes 16-byte accesses.
bool check_heads(const cpde_attention_shape& s, const cpde_heads* h, int tokens, int heads, bool output) {
    require(h, "null argument");
    if (!s.batch || !tokens) return true;
    require(h->data, "null tensor");
    require(h->batch >= 0 && h->token >= 0 && h->head >= 0, "negative stride");
    if (output) {
        // from the smallest stride up, each axis steps over all of the ones before
        std::pair<int64_t, int64_t> axes[3] = {{h->batch, s.batch}, {h->token, tokens}, {h->head, heads}};
        std::sort(axes, axes + 3);
        int64_t extent = s.head_dim;
        for (auto& [stride, count] : axes) {
            if (count == 1) continue;
            require(stride >= extent, "output elements overlap");
            extent = stride * (count - 1) + extent;
        }
    }
    const size_t size = type_bytes(s.dtype);
    // (a tile's rows are addressed with 32 bits)
    return wide(h->data, h->batch, size) && wide(h->data, h->token, size) && wide(h->data, h->head, size) &&
           s.head_dim * size % 16 == 0 && h->token * int64_t(size) < (int64_t(1) << 24);
}

AttentionArgs arguments(const Attention& p, const int* query_lengths, const int* key_lengths) {
    const auto& s = p.shape;
    const Cut& c = p.cut;
    AttentionArgs a{};
    a.query_lengths = query_lengths;
    a.key_lengths = key_lengths;
    a.pairs = s.batch * s.kv_heads;
    a.kv_heads = s.kv_heads;
    a.group = s.heads / s.kv_heads;
    a.queries = s.query_tokens;
    a.keys = s.key_tokens;
    a.dim = s.head_dim;
    a.left = s.left;
    a.right = s.right;
    a.scale = s.scale;
    a.scale2 = s.scale * kLog2e;
    a.span = c.span;
    a.row_lse = p.work;
    a.row_delta = p.work + c.stats / 2;
    a.part = p.work + c.stats;
    a.part_stats = a.part + c.part;
    a.key_part = a.part_stats + c.part_stats;
    return a;
}

int join_teams(int splits) {
    int teams = 1;
    while (teams < 8 && 2 * teams < splits) teams *= 2;
    return teams;
}
Join join_of(const float* part, const HeadView& out, int pairs, int splits, int rows, int group, float scale) {
    Join j{part, out, splits, rows, group, 0, join_teams(splits), scale};
    j.blocks = splits > 1 ? ceil_div(int64_t(pairs) * rows, 8 / j.teams) : 0;
    return j;
}
template <class T>
void join(Device& d, const AttentionArgs& a, std::initializer_list<Join> joins, const float* stats, float* lse) {
    JoinArgs j{};
    int n = 0, blocks = 0;
    for (const Join& one : joins) {
        j.joins[n++] = one;
        blocks += one.blocks;
    }
    if (!blocks) return;
    j.stats = stats;
    j.lse = lse;
    j.pairs = a.pairs;
    j.dim = a.dim;
    j.kv_heads = a.kv_heads;
    j.wide_part = a.dim % 4 == 0;
    j.wide_out = a.wide_out;
    hipLaunchKernelGGL((attention_join_k<T>), unsigned(blocks), 256, 0, d.stream, j);
}

template <class F>
void with_width(int dim, F body) {
    if (dim <= 32) body(std::integral_constant<int, 32>{});
    else if (dim <= 64) body(std::integral_constant<int, 64>{});
    else if (dim <= 96) body(std::integral_constant<int, 96>{});
    else body(std::integral_constant<int, 128>{});
}

template <class T>
void step(Device& d, const AttentionArgs& a, int rows, bool brief) {
    const unsigned blocks = unsigned(a.pairs) * unsigned(a.splits);
    const auto launch = [&](auto lanes, auto most, auto waves) {
        constexpr int kWaves = decltype(waves)::value;
        hipLaunchKernelGGL((attention_step_k<T, decltype(lanes)::value, decltype(most)::value, kWaves>), blocks,
                           64 * kWaves, 0, d.stream, a);
    };
    const auto with_waves = [&](auto lanes, auto most) {
        if (brief) launch(lanes, most, std::integral_constant<int, 16>{});
        else if constexpr (sizeof(T) == 4) launch(lanes, most, std::integral_constant<int, 4>{});
    };
    const auto with_rows = [&](auto lanes) {
        if (rows == 1) with_waves(lanes, std::integral_constant<int, 1>{});
        else with_waves(lanes, std::integral_constant<int, 2>{});
    };
    const int lanes = step_lanes(a.dim);
    if (lanes == 4) with_rows(std::integral_constant<int, 4>{});
    else if (lanes == 8) with_rows(std::integral_constant<int, 8>{});
    else with_rows(std::integral_constant<int, 16>{});
}

}  // namespace
}  // namespace cpde

struct cpde_attention_s : cpde::Attention {};
using namespace cpde;

extern "C" {

int cpde_attention_create(cpde_device* dev, const cpde_attention_shape* shape, cpde_attention** out) {
    return guarded([&] {
        require(dev && shape && out, "null argument");
        *out = nullptr;
        cpde_attention_shape s = *shape;
        check_dtype(s.dtype);
        require(s.batch >= 0 && s.query_tokens >= 0 && s.key_tokens >= 0, "negative size");
        require(s.heads >= 1 && s.kv_heads >= 1 && s.heads % s.kv_heads == 0,
                "query heads are a whole number of times the key heads");
        require(s.head_dim >= 1 && s.head_dim <= kMaxHeadDim, "a head is 1 to 128 wide");
        // (the backward divides by it, the forward takes it times log2 e)
        require(s.scale == 0 || (s.scale >= 1e-30f && s.scale <= 1e30f), "the scale is positive, or 0 for 1/sqrt(head_dim)");
        constexpr int64_t kMost = int64_t(1) << 30;  // (row and key numbers, and sums of two, stay inside 32 bits)
        require(int64_t(s.query_tokens) * (s.heads / s.kv_heads) <= kMost && s.key_tokens <= kMost, "too many tokens");
        if (s.scale == 0) s.scale = 1.f / std::sqrt(float(s.head_dim));
        s.left = s.left < 0 ? -1 : int(std::min<int64_t>(s.left, kMost - 2));
        s.right = s.right < 0 ? -1 : int(std::min<int64_t>(s.right, kMost - 2));
        require(!dev->capturing, "a capture is open on this device");
        auto p = std::make_unique<cpde_attention_s>();
        p->dev = dev;
        p->shape = s;
        p->seen = double(s.batch) * s.heads * seen_pairs(s);
        cut_launches(*p);
        const Cut& c = p->cut;
        const int64_t pairs = int64_t(s.batch) * s.kv_heads;
        // lanes of the largest launch (the runtime takes fewer than 2^32): forward, gradient, joins
        const int64_t forward = (c.step ? 1 : c.few ? ceil_div(c.rows, kWaveRows) : c.row_tiles) * int64_t(c.forward) *
                                (c.step && c.brief ? 1024 : 256);
        const int64_t gradient = c.few_gradient ? ceil_div(s.key_tokens, kWaveRows) + int64_t(ceil_div(c.rows, kWaveRows))
                                                : c.key_tiles * int64_t(c.key) + c.row_tiles * int64_t(c.query);
        const auto joined = [](int splits, int64_t rows) { return splits > 1 ? rows * 32 * join_teams(splits) : 0; };
        const int64_t joins = std::max(joined(c.forward, c.rows), joined(c.query, c.rows) + 2 * joined(c.key, s.key_tokens));
        const int64_t most = std::max({forward, s.backward ? gradient * 256 : 0, joins});
        // (with room for the last workgroup of each join)
        require(pairs <= kMost && (!pairs || most <= ((int64_t(1) << 32) - 1024) / pairs), "too many workgroups: split the batch");
        HIP_CHECK(hipMalloc(&p->work, std::max<size_t>(c.floats, 64) * sizeof(float)));
        *out = p.release();
    });
}

int cpde_attention_destroy(cpde_attention* attention) {
    return guarded([&] {
        if (!attention) return;
        sync_stream(*attention->dev, __LINE__);
        ++attention->dev->layout;
        HIP_CHECK(hipFree(attention->work));
        delete attention;
    });
}

int cpde_attention_info(cpde_attention* attention, char* text, size_t capacity) {
    return guarded([&] {
        require(attention && text && capacity, "null argument");
        const Cut& c = attention->cut;
        std::string s = std::string("forward attention_") + (c.step ? "step_k" : c.few ? "rows_k" : "forward_k") + " splits " +
                        std::to_string(c.forward);
        if (attention->shape.backward)
            s += std::string(", gradient attention_") + (c.few_gradient ? "few_gradient_k" : "gradient_k") + " key splits " +
                 std::to_string(c.key) + " query splits " + std::to_string(c.query);
        std::snprintf(text, capacity, "%s", s.c_str());
    });
}

int cpde_attention_forward(cpde_attention* attention, const cpde_heads* q, const cpde_heads* k, const cpde_heads* v,
                           const cpde_heads* out, float* lse, const int32_t* query_lengths,
                           const int32_t* key_lengths) {
    return guarded([&] {
        require(attention, "null argument");
        const Attention& p = *attention;
        const auto& s = p.shape;
        const Cut& c = p.cut;
        AttentionArgs a = arguments(p, query_lengths, key_lengths);
        const bool wq = check_heads(s, q, s.query_tokens, s.heads, false);
        const bool wk = check_heads(s, k, s.key_tokens, s.kv_heads, false);
        const bool wv = check_heads(s, v, s.key_tokens, s.kv_heads, false);
        a.wide_in = wq && wk && wv;
        a.wide_out = check_heads(s, out, s.query_tokens, s.heads, true);
        if (!a.pairs || !c.rows) return;
        a.q = view(*q);
        a.k = view(*k);
        a.v = view(*v);
        a.out = view(*out);
        a.lse = lse;
        a.splits = c.forward;
        a.tiles = c.row_tiles;
        Device& d = *p.dev;
        flush_reduce(d);
        TraceScope trace(d, kTraceAttention, 4.0 * p.seen * s.head_dim);
        with_type(s.dtype, [&](auto element) {
            using T = decltype(element);
            if (c.step) step<T>(d, a, c.rows, c.brief);
            else
                with_width(a.dim, [&](auto width) {
                    if (c.few) {
                        constexpr int DP = decltype(width)::value;
                        a.tiles = ceil_div(c.rows, kWaveRows);
                        hipLaunchKernelGGL((attention_rows_k<T, DP>), unsigned(a.pairs) * a.tiles * a.splits,
                                           (64 * kRowWaves<T, DP>), 0, d.stream, a);
                        return;
                    }
                    hipLaunchKernelGGL((attention_forward_k<T, decltype(width)::value>),
                                       unsigned(a.pairs) * a.tiles * a.splits, 256, 0, d.stream, a);
                });
            HIP_CHECK(hipGetLastError());
            join<T>(d, a, {join_of(a.part, a.out, a.pairs, a.splits, c.rows, a.group, 1.f)}, a.part_stats, lse);
        });
        HIP_CHECK(hipGetLastError());
    });
}

int cpde_attention_backward(cpde_attention* attention, const cpde_heads* q, const cpde_heads* k, const cpde_heads* v,
                            const cpde_heads* out, const float* lse, const cpde_heads* dout, const cpde_heads* dq,
                            const cpde_heads* dk, const cpde_heads* dv, const int32_t* query_lengths,
                            const int32_t* key_lengths) {
    return guarded([&] {
        require(attention, "null argument");
        const Attention& p = *attention;
        const auto& s = p.shape;
        require(s.backward, "the attention was created without a backward");
        const Cut& c = p.cut;
        AttentionArgs a = arguments(p, query_lengths, key_lengths);
        const bool in[] = {check_heads(s, q, s.query_tokens, s.heads, false),
                           check_heads(s, k, s.key_tokens, s.kv_heads, false),
                           check_heads(s, v, s.key_tokens, s.kv_heads, false),
                           check_heads(s, out, s.query_tokens, s.heads, false),
                           check_heads(s, dout, s.query_tokens, s.heads, false)};
        const bool to[] = {check_heads(s, dq, s.query_tokens, s.heads, true),
                           check_heads(s, dk, s.key_tokens, s.kv_heads, true),
                           check_heads(s, dv, s.key_tokens, s.kv_heads, true)};
        require(lse || !a.pairs || !c.rows, "null statistics");
        a.wide_in = in[0] && in[1] && in[2] && in[3] && in[4];
        a.wide_out = to[0] && to[1] && to[2];
        a.q = view(*q);
        a.k = view(*k);
        a.v = view(*v);
        a.out = view(*out);
        a.dout = view(*dout);
        a.dq = view(*dq);
        a.dk = view(*dk);
        a.dv = view(*dv);
        a.lse = const_cast<float*>(lse);
        if (!a.pairs) return;
        Device& d = *p.dev;
        flush_reduce(d);
        TraceScope trace(d, kTraceAttentionGradient, 10.0 * p.seen * s.head_dim);
        with_type(s.dtype, [&](auto element) {
            using T = decltype(element);
            const int64_t count = int64_t(s.batch) * s.heads * s.query_tokens;
            constexpr int64_t kAtOnce = int64_t(1) << 27;  // (a launch takes fewer than 2^32 lanes)
            for (int64_t first = 0; first < count; first += kAtOnce)
                hipLaunchKernelGGL((attention_delta_k<T>), unsigned((std::min(count - first, kAtOnce) + 15) / 16), 256, 0,
                                   d.stream, a, first);
            HIP_CHECK(hipGetLastError());
            a.tiles = c.row_tiles;
            a.splits = c.query;
            a.key_tiles = c.key_tiles;
            a.key_splits = c.key;
            if (c.few_gradient) {
                a.tiles = ceil_div(c.rows, kWaveRows);
                a.key_tiles = ceil_div(s.key_tokens, kWaveRows);
            }
            a.key_blocks = a.pairs * a.key_tiles * c.key;
            const unsigned blocks = unsigned(a.key_blocks) + unsigned(a.pairs) * unsigned(a.tiles * c.query);
            if (!blocks) return;
            with_width(a.dim, [&](auto width) {
                constexpr int DP = decltype(width)::value;
                if (c.few_gradient) hipLaunchKernelGGL((attention_few_gradient_k<T, DP>), blocks, 256, 0, d.stream, a);
                else hipLaunchKernelGGL((attention_gradient_k<T, DP>), blocks, 256, 0, d.stream, a);
            });
            HIP_CHECK(hipGetLastError());
            const float* second = a.key_part + size_t(c.key) * a.pairs * s.key_tokens * s.head_dim;
            join<T>(d, a,
                    {join_of(a.key_part, a.dk, a.pairs, c.key, s.key_tokens, 1, a.scale),
                     join_of(second, a.dv, a.pairs, c.key, s.key_tokens, 1, 1.f),
                     join_of(a.part, a.dq, a.pairs, c.query, c.rows, a.group, a.scale)},
                    nullptr, nullptr);
        });
        HIP_CHECK(hipGetLastError());
    });
}

}  // extern "C"
