// Rows of a table by token, scaled, and the table's gradient by sorted tokens.
#include "sequence.hpp"

namespace cpde {
namespace {

// Tokens up to which every workgroup looks for its rows' tokens itself (8,000 uneven ones
// of 1,000 rows x 32: 20 us, 51 sorted first), and up to which it does where there are no
// more workgroups than CUs, as a longer list leaves room for fewer (16,000 of 200 rows x
// 32: 38 us, 43 sorted; 16,384 of 20 rows x 200: 35 and 49; lists of 16,384 for all,
// 2,187 of 1,000 rows x 128: 15 us, 11 with lists of 8,192 then).
constexpr int kShort = 8192, kLong = 16384;
// And their rows' bytes in a workgroup's columns, as one row may have all of them (in 4
// MB, not in 2: 4,096 tokens of 3,000 rows x 512 15 us, 33 sorted; of 1,000 x 1,023 29
// and 41; but of 20,000 x 1,024 55 and 52).
constexpr int64_t kShortBytes = 4 << 20;
constexpr int kShortRows = 256;      // table rows of such a workgroup, at most
constexpr int kDigitBits = 10;       // at most, of one pass of the sort
constexpr int kSortTokens = 1024;    // per workgroup of such a pass
constexpr uint32_t kFan = 32;             // sorted tokens of a partial sum, and partial sums of one of the second level

struct Embedding {
    Device* dev = nullptr;
    int dtype = 0, rows = 0, width = 0, index_bytes = 0;
    int64_t tokens = 0;
    char* work = nullptr;  // of the gradient, see layout()
};

// The gradient's workspace.
struct Layout {
    size_t keys[2], places[2], counts, totals, sums1, sums2, bytes;
};
int bit_width(uint32_t v) {
    int bits = 0;
    while (v) v >>= 1, ++bits;
    return bits;
}
int sort_passes(int rows) { return (bit_width(uint32_t(rows)) + kDigitBits - 1) / kDigitBits; }
int digit_bits(int rows) { return (bit_width(uint32_t(rows)) + sort_passes(rows) - 1) / sort_passes(rows); }

Layout layout(const Embedding& e) {
    Layout l{};
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t begin = at;
        at += (bytes + 255) / 256 * 256;
        return begin;
    };
    const size_t n = size_t(e.tokens);
    for (int i = 0; i < 2; ++i) {
        l.keys[i] = take(4 * n);
        l.places[i] = take(4 * n);
    }
    l.counts = take(4 * ((n + kSortTokens - 1) / kSortTokens << digit_bits(e.rows)));
    l.totals = take(4 << kDigitBits);
    l.sums1 = take(4 * (n / kFan) * size_t(e.width));
    l.sums2 = take(4 * (n / (kFan * kFan)) * size_t(e.width));
    l.bytes = std::max<size_t>(at, 256);
    return l;
}

// An id as a sort key: ids outside the table sort behind every row.
template <class I>
__device__ inline uint32_t key_of(I id, int rows) {
    return id >= 0 && id < I(rows) ? uint32_t(id) : uint32_t(rows);
}

// Eight values of 16 bits, or four floats, of a row as floats: in one load where
// the rows are aligned, else one by one; values at or past `left` are zeros.
template <class T>
constexpr int kLane = 16 / sizeof(T);
template <class T>
__device__ inline void load_lane(float* v, const T* p, int64_t left, bool aligned) {
    if (aligned) {
        const vec<T, kLane<T>> in = *reinterpret_cast<const vec<T, kLane<T>>*>(p);
#pragma unroll
        for (int j = 0; j < kLane<T>; ++j) v[j] = float(in[j]);
    } else {
#pragma unroll
        for (int j = 0; j < kLane<T>; ++j) v[j] = j < left ? float(p[j]) : 0.f;
    }
}

// ---- lookup ---------------------------------------------------------------------------
// A lane copies 16 bytes of each of two rows, so that two ids and then two rows
// are under way.  Bound: HBM (the rows written; rows of common tokens come from the
// caches, which the rows written pass by: 32,768 uneven tokens of 1,024 16-bit values
// 19 us, 34 where they do not, 25 with one row a lane, 24 with four).
template <class T, class I>
__global__ __launch_bounds__(256) void embedding_lookup_k(const I* ids, uint64_t lanes, uint32_t per_row, const T* table,
                                                          int64_t table_stride, int rows, int width, float scale, T* out,
                                                          int64_t out_stride, bool aligned) {
    constexpr int N = kLane<T>, kDeep = 2;
    const uint64_t step = uint64_t(gridDim.x) * 256;
    for (uint64_t first = uint64_t(blockIdx.x) * 256 + threadIdx.x; first < lanes; first += kDeep * step) {
        uint64_t token[kDeep];
        uint32_t row[kDeep];
        int column[kDeep];
        float v[kDeep][N];
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
            const uint64_t i = first + u * step;
            token[u] = lanes <= 0xffffffffull ? uint32_t(i) / per_row : i / per_row;
            column[u] = int(i - token[u] * per_row) * N;
            row[u] = i < lanes ? key_of(ids[token[u]], rows) : uint32_t(rows);
        }
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
#pragma unroll
            for (int j = 0; j < N; ++j) v[u][j] = 0.f;
            if (row[u] < uint32_t(rows))
                load_lane(v[u], table + int64_t(row[u]) * table_stride + column[u], width - column[u], aligned);
        }
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
            if (first + u * step >= lanes) break;
            T* to = out + int64_t(token[u]) * out_stride + column[u];
            if (aligned) {
                vec<T, N> o;
#pragma unroll
                for (int j = 0; j < N; ++j) o[j] = T(v[u][j] * scale);
                __builtin_nontemporal_store(__builtin_bit_cast(u32x4, o), reinterpret_cast<u32x4*>(to));
            } else {
                for (int j = 0; j < N && column[u] + j < width; ++j) to[j] = T(v[u][j] * scale);
            }
        }
    }
}

// ---- sorting tokens by row ------------------------------------------------------------
// A stable radix sort of (row, place) pairs, so that a row's tokens stay in order.
// Lanes of a wave with the same digit find one another by one ballot a bit; the
// first of them takes their places from the wave's counter of that digit.
__device__ inline uint64_t same_digit(uint32_t digit, int bits, bool live) {
    uint64_t peers = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const bool set = (digit >> b) & 1;
        const uint64_t with = __ballot(set);
        peers &= set ? with : ~with;
    }
    return peers;
}
__device__ inline int take_place(int* counter, uint64_t peers, int lane) {
    const int first = __ffsll(static_cast<unsigned long long>(peers)) - 1;
    int base = 0;
    if (lane == first) base = atomicAdd(counter, __popcll(peers));
    return __shfl(base, first) + __popcll(peers & ((1ull << lane) - 1));
}

// Per pass, the digits of every 1,024 tokens counted, the counts'
// running sums over those blocks (one wave a digit), and the pairs moved.  `ids` is
// null after the first pass.
template <class I>
__global__ __launch_bounds__(256) void embedding_count_k(const I* ids, const uint32_t* keys, uint32_t tokens, int rows,
                                                         int shift, int bits, int* counts) {
    __shared__ int counter[1 << kDigitBits];
    const int bins = 1 << bits;
    for (int b = threadIdx.x; b < bins; b += 256) counter[b] = 0;
    __syncthreads();
    const uint32_t begin = blockIdx.x * uint32_t(kSortTokens) + threadIdx.x;
#pragma unroll
    for (uint32_t j = 0; j < kSortTokens; j += 256)
        if (begin + j < tokens)
            atomicAdd(&counter[((ids ? key_of(ids[begin + j], rows) : keys[begin + j]) >> shift) & (bins - 1)], 1);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 256) counts[size_t(b) * gridDim.x + blockIdx.x] = counter[b];
}

// counts[digit][block] to sums over the blocks before, totals[digit] the whole row.
__global__ __launch_bounds__(256) void embedding_scan_k(int* counts, int* totals, int bins, uint32_t blocks) {
    const int lane = threadIdx.x & 63, bin = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (bin >= bins) return;
    int* row = counts + size_t(bin) * blocks;
    int carry = 0;
    for (uint32_t first = 0; first < blocks; first += 64) {
        const uint32_t i = first + lane;
        const int value = i < blocks ? row[i] : 0;
        int sum = value;
        for (int d = 1; d < 64; d <<= 1) {
            const int other = __shfl_up(sum, d);
            if (lane >= d) sum += other;
        }
        if (i < blocks) row[i] = carry + sum - value;
        carry += __shfl(sum, 63);
    }
    if (lane == 0) totals[bin] = carry;
}

template <class I>
__global__ __launch_bounds__(256) void embedding_move_k(const I* ids, const uint32_t* keys, const uint32_t* places,
                                                        uint32_t tokens, int rows, int shift, int bits,
                                                        const int* counts, const int* totals, uint32_t* to_keys,
                                                        uint32_t* to_places) {
    __shared__ int counter[4][1 << kDigitBits];
    __shared__ int waves[4];
    const int bins = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int kRounds = kSortTokens / 256;  // of a wave's quarter
    constexpr int kBins = (1 << kDigitBits) / 256;
    for (int b = threadIdx.x; b < bins; b += 256)
        for (int w = 0; w < 4; ++w) counter[w][b] = 0;
    const uint32_t begin = blockIdx.x * uint32_t(kSortTokens) + wave * (kSortTokens / 4) + lane;
    uint32_t k[kRounds], p[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const uint32_t i = begin + r * 64;
        k[r] = i < tokens ? ids ? key_of(ids[i], rows) : keys[i] : 0;
        p[r] = i < tokens && !ids ? places[i] : i;
    }
    // a lane's digits are neighbours: kBins of them from kBins * thread
    int total[kBins], before[kBins], sum = 0;
#pragma unroll
    for (int j = 0; j < kBins; ++j) {
        const int b = threadIdx.x * kBins + j;
        total[j] = b < bins ? totals[b] : 0;
        before[j] = b < bins ? counts[size_t(b) * gridDim.x + blockIdx.x] : 0;
        sum += total[j];
    }
    int running = sum;
    for (int d = 1; d < 64; d <<= 1) {
        const int other = __shfl_up(running, d);
        if (lane >= d) running += other;
    }
    if (lane == 63) waves[wave] = running;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
        if (begin + r * 64 < tokens) atomicAdd(&counter[wave][(k[r] >> shift) & (bins - 1)], 1);
    __syncthreads();
    running -= sum;
    for (int w = 0; w < wave; ++w) running += waves[w];
#pragma unroll
    for (int j = 0; j < kBins; ++j) {
        const int b = threadIdx.x * kBins + j;
        if (b < bins) {
            int at = running + before[j];
            for (int w = 0; w < 4; ++w) {
                const int n = counter[w][b];
                counter[w][b] = at;
                at += n;
            }
        }
        running += total[j];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const bool live = begin + r * 64 < tokens;
        const uint32_t digit = (k[r] >> shift) & (bins - 1);
        const uint64_t peers = same_digit(digit, bits, live);
        if (live) {
            const int to = take_place(&counter[wave][digit], peers, lane);
            to_keys[to] = k[r];
            to_places[to] = p[r];
        }
    }
}

// ---- sums of sorted tokens ------------------------------------------------------------
struct SumArgs {
    const uint32_t *keys, *places;
    const void* dout;
    int64_t dout_stride;
    float* dtable;
    int64_t dtable_stride;
    float *sums1, *sums2;  // of whole runs of kFan and kFan^2 tokens, [run][width]
    uint32_t tokens;
    int rows, width, accumulate, group_rows, lanes;  // lanes a row of `width` takes in one slice (a power of two)
    float scale;
    bool aligned_out;
};

// Four floats of any alignment.
__device__ inline vec<float, 4> load_floats(const float* p) {
    vec<float, 4> v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// A lane's values of a partial sum, whose rows are `width` floats; those at or past
// `left` are zeros.
template <int N>
__device__ inline void load_sum(float* v, const float* p, int left, int width) {
    if (width % 4 == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const vec<float, 4> in = j < left ? load_floats(p + j) : vec<float, 4>{};
#pragma unroll
            for (int q = 0; q < 4; ++q) v[j + q] = in[q];
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < left ? p[j] : 0.f;
    }
}

// A lane's columns of dout: sixteen bytes of a row as they are in memory, by one load
// of any alignment; a row's last ones are the last of its last 16 bytes, moved down when
// they are added (a move behind the load would wait for it).  Rows shorter than that
// are read value by value.  Lanes past the width read the row's last bytes and are not
// used.
// The form is a template's, as a branch between two loads waits for the first (4,000
// tokens of 400 rows x 1,023 in 16 bits 26 us, 52 with branches; 131,072 of 65,536 x 512
// 116 and 125).
template <class T, bool WIDE>
struct Columns {
    static constexpr int N = kLane<T>;
    const T* base;
    int64_t stride;
    int left, shift;  // values from the lane's column on; bits of the move
    bool moved;
    __device__ Columns(const SumArgs& a, int column) : stride(a.dout_stride), left(a.width - column) {
        moved = WIDE && a.width % N;
        const int back = WIDE ? std::max(0, N - left) : 0;
        shift = left > 0 ? back * int(sizeof(T)) * 8 : 0;
        base = static_cast<const T*>(a.dout) + column - back;
    }
    __device__ vec<T, N> load(int64_t token) const {
        const T* p = base + token * stride;
        vec<T, N> v = {};
        if constexpr (WIDE) {
            __builtin_memcpy(&v, p, 16);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (j < left) v[j] = p[j];
        }
        return v;
    }
    __device__ void add(float* acc, vec<T, N> v) const {
        if (moved) {
            unsigned __int128 bits;
            __builtin_memcpy(&bits, &v, 16);
            bits >>= shift;
            __builtin_memcpy(&v, &bits, 16);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += float(v[j]);
    }
};

// Partial sums of the aligned runs of kFan tokens that lie whole inside one row: a
// common token's row is then the sum of few terms, whatever its count.  A group of
// lanes a run, so that a common token's runs spread over the device.
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void embedding_partial_k(SumArgs a, uint32_t runs) {
    constexpr int N = kLane<T>;
    const uint64_t run = (uint64_t(blockIdx.x) * 256 + threadIdx.x) / unsigned(a.lanes);
    const int column = (blockIdx.y * a.lanes + (threadIdx.x & (a.lanes - 1))) * N, left = a.width - column;
    if (run >= runs || left <= 0) return;
    const uint32_t first = uint32_t(run) * kFan, row = a.keys[first];
    if (row >= uint32_t(a.rows) || row != a.keys[first + kFan - 1]) return;
    const Columns<T, WIDE> columns(a, column);
    float acc[N] = {};
#pragma unroll 1
    for (uint32_t i = 0; i < kFan; i += 16) {
        uint32_t place[16];
        vec<T, N> v[16];
#pragma unroll
        for (uint32_t u = 0; u < 16; ++u) place[u] = a.places[first + i + u];
#pragma unroll
        for (uint32_t u = 0; u < 16; ++u)
            v[u] = columns.load(place[u]);
#pragma unroll
        for (int u = 0; u < 16; ++u) columns.add(acc, v[u]);
    }
    float* to = a.sums1 + size_t(run) * a.width + column;
    for (int j = 0; j < N && j < left; ++j) to[j] = acc[j];
}

// The same of kFan such runs; a workgroup each.
__global__ __launch_bounds__(256) void embedding_partial2_k(SumArgs a) {
    const uint32_t first = blockIdx.x * kFan * kFan, row = a.keys[first];
    if (row >= uint32_t(a.rows) || row != a.keys[first + kFan * kFan - 1]) return;
    for (int column = threadIdx.x; column < a.width; column += 256) {
        const float* from = a.sums1 + size_t(blockIdx.x) * kFan * a.width + column;
        float sum = 0;
#pragma unroll
        for (uint32_t r = 0; r < kFan; ++r) sum += from[size_t(r) * a.width];
        a.sums2[size_t(blockIdx.x) * a.width + column] = sum;
    }
}

// A lane's columns of one row of the table's gradient.
template <int N>
__device__ inline void write_row(const SumArgs& a, int64_t row, int column, const float* sum) {
    float* out = a.dtable + row * a.dtable_stride + column;
    const int left = a.width - column;
    if (a.aligned_out) {
        if (left > 0)
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                vec<float, 4>* p = reinterpret_cast<vec<float, 4>*>(out + j);
                vec<float, 4> v = {sum[j] * a.scale, sum[j + 1] * a.scale, sum[j + 2] * a.scale, sum[j + 3] * a.scale};
                if (a.accumulate) v += *p;
                __builtin_nontemporal_store(v, p);
            }
    } else {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            if (j + 4 <= left) {
                vec<float, 4> v = {sum[j] * a.scale, sum[j + 1] * a.scale, sum[j + 2] * a.scale, sum[j + 3] * a.scale};
                if (a.accumulate) v += load_floats(out + j);
                __builtin_memcpy(out + j, &v, 16);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (j + q < left) out[j + q] = (a.accumulate ? out[j + q] : 0.f) + sum[j + q] * a.scale;
            }
        }
    }
}

// Short lists, in one launch without a sort of the whole: a workgroup reads all ids
// and puts its rows' tokens into LDS by row (stably: counted, then moved, a wave each),
// and a group of lanes sums each row's, eight loads under way.  A row of more tokens
// than `alone` is shared by all groups, in shares by its tokens' order, joined in a
// tree.  Workgroups along y take slices of the columns.
template <class T, class I, int LIST, bool WIDE>
__global__ __launch_bounds__(256) void embedding_short_k(SumArgs a, const I* ids, int block_rows, int alone) {
    constexpr int N = kLane<T>, kRounds = 16;
    __shared__ uint16_t order[LIST];  // tokens by row
    __shared__ int counter[4][kShortRows], places[4][kShortRows], start[kShortRows + 1];
    __shared__ float shares[4 * 64 * N];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t first = blockIdx.x * block_rows;
    const int rows = int(std::min<uint32_t>(block_rows, a.rows - first));
    // wave w reads tokens [w * share, (w + 1) * share), in rounds of 64
    const int rounds = (a.tokens + 255) / 256, begin = wave * rounds * 64 + lane;
    uint32_t key[kRounds], some = 0;  // keys of 16 rounds; the rounds that have any of the workgroup's rows
    const auto load = [&](int from) {
        some = 0;
        uint64_t in[kRounds];
#pragma unroll
        for (int r = 0; r < kRounds; ++r)
            if (from + r < rounds) in[r] = uint64_t(int64_t(ids[std::min<uint32_t>(begin + (from + r) * 64, a.tokens - 1)]));
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            if (from + r >= rounds) continue;
            // (ids outside the table, too, are no less than `rows` from `first` on)
            const uint64_t row = in[r] - first;
            const bool live = row < uint32_t(rows) && begin + (from + r) * 64 < a.tokens;
            key[r] = live ? uint32_t(row) : kShortRows;
            if (__any(live)) some |= 1u << r;
        }
    };
    load(0);
#pragma unroll
    for (int w = 0; w < 4; ++w) counter[w][threadIdx.x] = 0;
    __syncthreads();
    for (int from = 0; from < rounds; from += kRounds) {
        if (from) load(from);
#pragma unroll
        for (int r = 0; r < kRounds; ++r)
            if (some >> r & 1 && key[r] < kShortRows) atomicAdd(&counter[wave][key[r]], 1);
    }
    __syncthreads();
    // (every wave makes the running sums for itself: no barrier before the move)
    for (int c = 0, carry = 0; c < rows; c += 64) {
        int n[4], tokens = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) tokens += n[w] = counter[w][c + lane];
        int before = tokens;
        for (int step = 1; step < 64; step <<= 1) {
            const int other = __shfl_up(before, step);
            if (lane >= step) before += other;
        }
        const int sum = __shfl(before, 63);
        before += carry - tokens;
        if (wave == 0) {
            start[c + lane] = before;
            if (lane == 63) start[c + 64] = before + tokens;
        }
#pragma unroll
        for (int w = 0; w < 3; ++w)
            if (w < wave) before += n[w];
        places[wave][c + lane] = before;
        carry += sum;
    }
    const int bits = block_rows > 1 ? 32 - __clz(block_rows - 1) : 0;
    for (int from = 0; from < rounds; from += kRounds) {
        if (rounds > kRounds) load(from);
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            if (!(some >> r & 1)) continue;
            const bool live = key[r] < kShortRows;
            const uint64_t peers = same_digit(key[r], bits, live);
            if (live) order[take_place(&places[wave][key[r]], peers, lane)] = uint16_t(begin + (from + r) * 64);
        }
    }
    __syncthreads();
    const int in = lane & (a.lanes - 1), group = threadIdx.x / a.lanes, groups = 256 / a.lanes;
    for (int slice = blockIdx.y; slice * a.lanes * N < a.width; slice += gridDim.y) {
        const int column = (slice * a.lanes + in) * N;
        const Columns<T, WIDE> columns(a, column);
        // acc += the tokens at [from, to) of the order
        const auto sum = [&](float* acc, int from, int to) {
            int p = from;
            for (; p + 8 <= to; p += 8) {
                vec<T, N> v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = columns.load(order[p + u]);
#pragma unroll
                for (int u = 0; u < 8; ++u) columns.add(acc, v[u]);
            }
            for (; p < to; p += 4) {
                vec<T, N> v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = columns.load(order[std::min(p + u, to - 1)]);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (p + u < to) columns.add(acc, v[u]);
            }
        };
        for (int r = group; r < rows; r += groups) {
            if (start[r + 1] - start[r] > alone) continue;
            float acc[N] = {};
            sum(acc, start[r], start[r + 1]);
            write_row<N>(a, first + r, column, acc);
        }
        for (int r = 0; r < rows; ++r) {
            const int tokens = start[r + 1] - start[r];
            if (tokens <= alone) continue;
            float acc[N] = {};
            sum(acc, start[r] + tokens * group / groups, start[r] + tokens * (group + 1) / groups);
            for (int step = a.lanes; step < 64; step <<= 1)
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] += __shfl_xor(acc[j], step);
            if (lane < a.lanes)
#pragma unroll
                for (int j = 0; j < N; ++j) shares[(wave * 64 + in) * N + j] = acc[j];
            __syncthreads();
            if (group == 0) {
                for (int w = 1; w < 4; ++w)
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] += shares[(w * 64 + in) * N + j];
                write_row<N>(a, first + r, column, acc);
            }
            __syncthreads();
        }
    }
}

// First sorted tokens whose rows are at least `row` and `end`, by a group of `lanes`
// lanes: each step probes `lanes` places of both searches at once.  All lanes of the
// wave take part.
__device__ inline void first_of(const uint32_t* keys, uint32_t tokens, uint32_t row, uint32_t end, int lanes,
                                uint32_t& first, uint32_t& last) {
    const int lane = threadIdx.x & 63, in = lane & (lanes - 1);
    const uint64_t group = (lanes == 64 ? ~0ull : (1ull << lanes) - 1) << (lane - in);
    uint32_t low[2] = {0, 0}, high[2] = {tokens, tokens};  // the answers lie in [low, high]
    const uint32_t want[2] = {row, end};
    while (__any(low[0] < high[0] || low[1] < high[1])) {
        uint32_t key[2];
        const auto probe = [&](int s, int i) {
            return low[s] + uint32_t((high[s] - low[s]) * uint64_t(i + 1) / uint64_t(lanes + 1));
        };
#pragma unroll
        for (int s = 0; s < 2; ++s) key[s] = low[s] < high[s] ? keys[probe(s, in)] : 0;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const bool open = low[s] < high[s];
            const int below = __popcll(__ballot(open && key[s] < want[s]) & group);  // probes 0..below-1 are less
            if (open) {
                const uint32_t to = below == lanes ? high[s] : probe(s, below);
                if (below) low[s] = probe(s, below - 1) + 1;
                high[s] = to;
            }
        }
    }
    first = low[0];
    last = low[1];
}

// The table's gradient: a group of lanes takes `group_rows` rows and their sorted
// tokens and writes each row once, the sum of its tokens (or zeros).  Tokens come
// `lanes` at a time, a lane each, and their rows of dout in eights, the next eight
// under way while one is added, whatever rows of the table they belong to.  Where a
// whole run of kFan tokens, or of kFan such runs, belongs to one row, its partial
// sum stands for it: the order of a sum depends on the tokens alone.  Bound: HBM
// (131,072 uneven tokens of 65,536 rows x 512, bf16: 69 us, 114 MB read and 165 written;
// the sort's 33 us and the partial sums' 20 come before; 115 the whole).
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void embedding_sum_k(SumArgs a) {
    constexpr int N = kLane<T>;
    const int lane = threadIdx.x & 63, in = lane & (a.lanes - 1), begin_lane = lane - in;
    const uint64_t mine = (a.lanes == 64 ? ~0ull : (1ull << a.lanes) - 1) << begin_lane;
    const uint64_t group = (uint64_t(blockIdx.x) * 256 + threadIdx.x) / unsigned(a.lanes);
    const int column = (blockIdx.y * a.lanes + in) * N, left = a.width - column;
    const uint64_t begin_row = std::min(group * uint64_t(a.group_rows), uint64_t(a.rows));
    const uint32_t end_row = uint32_t(std::min(begin_row + a.group_rows, uint64_t(a.rows)));
    uint32_t at, end;
    first_of(a.keys, a.tokens, uint32_t(begin_row), end_row, a.lanes, at, end);
    const Columns<T, WIDE> columns(a, column);
    uint32_t row = uint32_t(begin_row);
    float acc[N] = {};
    const auto finish_before = [&](uint32_t next) {
        for (; row < next; ++row) {
            write_row<N>(a, row, column, acc);
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = 0.f;
        }
    };
    while (at < end) {
        // the next tokens, a lane each, to the next place where a whole run may begin;
        // and, where one begins here, how many follow one another
        const uint32_t here = std::min(std::min(end - at, kFan - at % kFan), uint32_t(a.lanes));
        const uint32_t i = at + std::min(uint32_t(in), here - 1);
        const uint32_t my_key = a.keys[i], my_place = a.places[i];
        uint32_t span = 0;
        int runs = 0;
        if (at % kFan == 0 && at + kFan <= end) {
            const uint32_t key = __shfl(my_key, begin_lane);
            const auto follow = [&](uint32_t s) {
                const uint64_t last = uint64_t(at) + uint64_t(in + 1) * s;
                const uint64_t no = ~__ballot(last <= end && a.keys[last <= end ? last - 1 : at] == key) & mine;
                return no ? __ffsll(static_cast<unsigned long long>(no)) - 1 - begin_lane : a.lanes;
            };
            if (at % (kFan * kFan) == 0) {
                span = kFan * kFan;
                runs = follow(span);
            }
            if (!runs) {
                span = kFan;
                runs = follow(span);
            }
            if (runs) finish_before(key);
        }
        if (runs) {
            if (span == kFan)  // (up to where the second level may take over)
                runs = std::min(runs, int((kFan * kFan - at % (kFan * kFan)) / kFan));
            const float* sums = (span == kFan ? a.sums1 : a.sums2) + size_t(at / span) * a.width + column;
            constexpr int kSums = 32 / N;
            for (int r = 0; r < runs; r += kSums) {
                float v[kSums][N];
#pragma unroll
                for (int u = 0; u < kSums; ++u)
                    load_sum<N>(v[u], sums + size_t(std::min(r + u, runs - 1)) * a.width, left, a.width);
#pragma unroll
                for (int u = 0; u < kSums; ++u)
                    if (r + u < runs)
#pragma unroll
                        for (int j = 0; j < N; ++j) acc[j] += v[u][j];
            }
            at += runs * span;
            continue;
        }
        constexpr int kBatch = 8;
        vec<T, N> v[2][kBatch];
        const auto load = [&](vec<T, N>* to, uint32_t from) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const uint32_t place = __shfl(my_place, begin_lane + int(std::min(from + u, here - 1)));
                to[u] = columns.load(place);
            }
        };
        const auto add = [&](const vec<T, N>* from, uint32_t first) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const uint32_t key = __shfl(my_key, begin_lane + int(std::min(first + u, here - 1)));
                if (first + u < here) {
                    finish_before(key);
                    columns.add(acc, from[u]);
                }
            }
        };
        load(v[0], 0);
        for (uint32_t n = 0; n < here; n += 2 * kBatch) {
            if (n + kBatch < here) load(v[1], n + kBatch);
            add(v[0], n);
            if (n + 2 * kBatch < here) load(v[0], n + 2 * kBatch);
            if (n + kBatch < here) add(v[1], n + kBatch);
        }
        at += here;
    }
    finish_before(end_row);
}

template <class T, class I, bool WIDE>
void gradient(const Embedding& e, const I* ids, uint32_t tokens, SumArgs a) {
    Device& d = *e.dev;
    const Layout l = layout(e);
    const auto part = [&](size_t at) { return reinterpret_cast<uint32_t*>(e.work + at); };
    a.tokens = tokens;
    constexpr int N = kLane<T>;
    const int per_row = (e.width + N - 1) / N;
    a.lanes = 1;
    while (a.lanes < per_row && a.lanes < 64) a.lanes <<= 1;
    if (tokens <= kLong) {
        const int fill = 4 * d.compute_units;  // workgroups
        const int rows = int(std::clamp<int64_t>((int64_t(e.rows) + fill - 1) / fill, 1, kShortRows));
        const int blocks = (e.rows + rows - 1) / rows;
        // Tables of few rows: more workgroups by slices of the columns, of 64 bytes at
        // least; twice as many where the rows of common tokens are what takes the time
        // (4,000 tokens of 400 rows x 1,023: 26 us, 31 with `fill` ones; 2,187 of 1,000 x 128,
        // 1 MB: 7.1, 11.9 with twice as many).
        const int64_t bytes = int64_t(tokens) * e.width * int64_t(sizeof(T));
        const int wanted = bytes > 2 << 20 ? 2 * fill : fill;
        int lanes = a.lanes;
        const auto slices = [&] { return 2 * blocks <= wanted ? std::min((per_row + lanes - 1) / lanes, 65535) : 1; };
        while (lanes > 4 && 2 * int64_t(blocks) * slices() <= wanted) lanes >>= 1;
        if ((tokens <= kShort || blocks * slices() <= d.compute_units) &&
            bytes <= kShortBytes * slices()) {
            a.lanes = lanes;
            const auto kernel = tokens <= kShort ? embedding_short_k<T, I, kShort, WIDE> : embedding_short_k<T, I, kLong, WIDE>;
            // (few rows a workgroup leave groups of lanes idle, so shorter ones are shared: 242
            // tokens of 11 rows x 344 5.3 us, 6.9 where rows of up to 32 tokens are not)
            hipLaunchKernelGGL(kernel, dim3(blocks, slices()), 256, 0, d.stream, a, ids, rows, rows > 4 ? 32 : 8);
            return;
        }
    }
    const int digit = digit_bits(e.rows), passes = sort_passes(e.rows);
    const unsigned blocks = (tokens + kSortTokens - 1) / kSortTokens;
    int *counts = reinterpret_cast<int*>(e.work + l.counts), *totals = reinterpret_cast<int*>(e.work + l.totals);
    int now = 0;
    for (int p = 0; p < passes; ++p) {
        const I* source = p ? nullptr : ids;
        hipLaunchKernelGGL((embedding_count_k<I>), blocks, 256, 0, d.stream, source, part(l.keys[now]), tokens, e.rows,
                           p * digit, digit, counts);
        hipLaunchKernelGGL(embedding_scan_k, ((1u << digit) + 3) / 4, 256, 0, d.stream, counts, totals, 1 << digit, blocks);
        hipLaunchKernelGGL((embedding_move_k<I>), blocks, 256, 0, d.stream, source, part(l.keys[now]), part(l.places[now]),
                           tokens, e.rows, p * digit, digit, counts, totals, part(l.keys[1 - now]), part(l.places[1 - now]));
        now = 1 - now;
    }
    a.keys = part(l.keys[now]);
    a.places = part(l.places[now]);
    a.sums1 = reinterpret_cast<float*>(part(l.sums1));
    a.sums2 = reinterpret_cast<float*>(part(l.sums2));
    const unsigned slices = unsigned((per_row + a.lanes - 1) / a.lanes);
    const uint32_t runs = tokens / kFan;
    if (runs)
        hipLaunchKernelGGL((embedding_partial_k<T, WIDE>), dim3(unsigned((uint64_t(runs) * a.lanes + 255) / 256), slices), 256, 0,
                           d.stream, a, runs);
    if (runs / kFan) hipLaunchKernelGGL(embedding_partial2_k, runs / kFan, 256, 0, d.stream, a);
    // A group's lanes also look through the tokens, so narrow rows have idle ones (60,000
    // tokens of 20 rows x 8: 59 us with 16 lanes, 64 with 8; 30,000 of 64 x 32 72 and 87).
    a.lanes = std::max(a.lanes, 16);
    // Rows a group: enough that a search serves several, few enough that common tokens
    // do not hold a wave back (131,072 uneven tokens of 65,536 rows x 512: 4 rows 116 us, 2
    // rows 127, 8 rows 129).
    const int64_t groups_wanted = int64_t(d.compute_units) * 64 / slices;
    a.group_rows = int(std::clamp<int64_t>(e.rows / std::max<int64_t>(groups_wanted, 1), 1, 16));
    const uint64_t groups = (uint64_t(e.rows) + a.group_rows - 1) / a.group_rows;
    hipLaunchKernelGGL((embedding_sum_k<T, WIDE>), dim3(unsigned((groups * unsigned(a.lanes) + 255) / 256), slices), 256, 0, d.stream, a);
}

void check_rows(const cpde_rows* r, int64_t count, int width, bool output) {
    require(r, "null argument");
    require(r->data || count == 0, "null tensor");
    require(r->stride >= 0, "negative stride");
    require(!output || count <= 1 || r->stride >= width, "output rows overlap");
}

}  // namespace
}  // namespace cpde

struct cpde_embedding_s : cpde::Embedding {};
using namespace cpde;

extern "C" {

int cpde_embedding_create(cpde_device* dev, int dtype, int rows, int width, int64_t tokens, int index_bytes,
                          cpde_embedding** out) {
    return guarded([&] {
        require(dev && out, "null argument");
        *out = nullptr;
        check_dtype(dtype);
        require(rows >= 1 && rows < (1 << 30) && width >= 1 && width <= (1 << 22), "invalid table size");
        require(tokens >= 0 && tokens < (int64_t(1) << 31) - kSortTokens, "invalid token count");
        require(index_bytes == 4 || index_bytes == 8, "ids are 4 or 8 bytes");
        auto e = std::make_unique<cpde_embedding_s>();
        e->dev = dev;
        e->dtype = dtype;
        e->rows = rows;
        e->width = width;
        e->tokens = tokens;
        e->index_bytes = index_bytes;
        require(!dev->capturing, "a capture is open on this device");
        HIP_CHECK(hipMalloc(&e->work, layout(*e).bytes));
        *out = e.release();
    });
}

int cpde_embedding_destroy(cpde_embedding* embedding) {
    return guarded([&] {
        if (!embedding) return;
        sync_stream(*embedding->dev, __LINE__);
        ++embedding->dev->layout;
        HIP_CHECK(hipFree(embedding->work));
        delete embedding;
    });
}

int cpde_embedding_forward(cpde_embedding* embedding, const void* ids, int64_t tokens, const cpde_rows* table,
                           float scale, const cpde_rows* out) {
    return guarded([&] {
        require(embedding, "null argument");
        const Embedding& e = *embedding;
        require(tokens >= 0 && tokens <= e.tokens, "more tokens than the embedding was created for");
        require(ids || tokens == 0, "null tensor");
        check_rows(table, e.rows, e.width, false);
        check_rows(out, tokens, e.width, true);
        if (!tokens) return;
        const size_t size = type_bytes(e.dtype);
        const bool aligned = wide(table->data, table->stride, size) && wide(out->data, out->stride, size) &&
                             e.width * size % 16 == 0;
        flush_reduce(*e.dev);
        TraceScope trace(*e.dev, kTraceEmbedding, double(tokens) * (2.0 * e.width * double(size) + e.index_bytes));
        with_type(e.dtype, [&](auto element) {
            using T = decltype(element);
            const uint32_t per_row = uint32_t((e.width + kLane<T> - 1) / kLane<T>);
            const uint64_t lanes = uint64_t(tokens) * per_row;
            const unsigned blocks =
                unsigned(std::min<uint64_t>((lanes + 255) / 256, uint64_t(e.dev->compute_units) * 64));
            const auto launch = [&](auto* at) {
                using I = std::remove_const_t<std::remove_pointer_t<decltype(at)>>;
                hipLaunchKernelGGL((embedding_lookup_k<T, I>), blocks, 256, 0, e.dev->stream, at, lanes, per_row,
                                   static_cast<const T*>(table->data), table->stride, e.rows, e.width, scale,
                                   static_cast<T*>(out->data), out->stride, aligned);
            };
            if (e.index_bytes == 4) launch(static_cast<const int32_t*>(ids));
            else launch(static_cast<const int64_t*>(ids));
        });
        HIP_CHECK(hipGetLastError());
    });
}

int cpde_embedding_backward(cpde_embedding* embedding, const void* ids, int64_t tokens, const cpde_rows* dout,
                            float scale, const cpde_rows* dtable, int accumulate) {
    return guarded([&] {
        require(embedding, "null argument");
        const Embedding& e = *embedding;
        require(tokens >= 0 && tokens <= e.tokens, "more tokens than the embedding was created for");
        require(ids || tokens == 0, "null tensor");
        check_rows(dout, tokens, e.width, false);
        check_rows(dtable, e.rows, e.width, true);
        const size_t size = type_bytes(e.dtype);
        SumArgs a{};
        a.dout = dout->data;
        a.dout_stride = dout->stride;
        a.dtable = static_cast<float*>(dtable->data);
        a.dtable_stride = dtable->stride;
        a.rows = e.rows;
        a.width = e.width;
        a.accumulate = accumulate != 0;
        a.scale = scale;
        a.aligned_out = wide(dtable->data, dtable->stride, 4) && e.width * size % 16 == 0;
        flush_reduce(*e.dev);
        TraceScope trace(*e.dev, kTraceEmbedding,
                         double(tokens) * (double(size) * e.width + e.index_bytes) + 4.0 * e.rows * double(e.width));
        with_type(e.dtype, [&](auto element) {
            using T = decltype(element);
            const auto run = [&](auto wide) {
                constexpr bool WIDE = decltype(wide)::value;
                if (e.index_bytes == 4) gradient<T, int32_t, WIDE>(e, static_cast<const int32_t*>(ids), uint32_t(tokens), a);
                else gradient<T, int64_t, WIDE>(e, static_cast<const int64_t*>(ids), uint32_t(tokens), a);
            };
            if (e.width >= kLane<T>) run(std::true_type{});
            else run(std::false_type{});
        });
        HIP_CHECK(hipGetLastError());
    });
}

}  // extern "C"
