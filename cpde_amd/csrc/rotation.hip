// Queries and keys on their way from their products into attention: each head's vector
// divided by its root mean square, times a weight a column, and its pairs of columns
// turned by an angle that goes with the token's position.
#include <cmath>

#include "sequence.hpp"

namespace cpde {
namespace {

constexpr int kMaxDim = 256;

struct Rotation {
    Device* dev = nullptr;
    cpde_rotation_shape shape{};
    double* rates = nullptr;  // turns a position of each pair
    float* part = nullptr;    // weight gradients of the workgroups, [workgroup][queries, keys][dim]
    int blocks = 0;           // of the gradient
};

// One side, queries or keys.
struct Side {
    const char* x;
    char* y;         // forward: the result; gradient: dx
    const char* dy;
    const char* weight;
    int64_t x_batch, x_token, x_head, y_batch, y_token, y_head, dy_batch, dy_token, dy_head;
    int heads;
};
struct RotationArgs {
    Side side[2];
    const double* rates;
    const int* positions;
    float* part;
    int64_t count;  // tokens of all entries
    int tokens, dim, pairs, interleaved, norm;
    int most;  // tokens of a workgroup at once, at most kTokens
    float eps;
};
constexpr int kTokens = 16;

// Sum over groups of LANES neighbouring lanes, each the whole sum.
template <int LANES>
__device__ inline float sum_group(float x) {
    const auto move = [](float v, auto control) {
        return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), decltype(control)::value, 0xf, 0xf, true));
    };
    x += move(x, std::integral_constant<int, 0xB1>{});                    // quad_perm [1,0,3,2]
    x += move(x, std::integral_constant<int, 0x4E>{});                    // quad_perm [2,3,0,1]
    if (LANES >= 8) x += move(x, std::integral_constant<int, 0x141>{});   // row_half_mirror
    if (LANES >= 16) x += move(x, std::integral_constant<int, 0x140>{});  // row_mirror
    if (LANES >= 32) x += __shfl_xor(x, 16);
    if (LANES >= 64) x += __shfl_xor(x, 32);
    return x;
}

// What a lane holds of a head's vector: pairs of columns.  WIDE: four of them, as two runs of
// four columns, from `first` and from `second` (interleaved: one run of eight); otherwise two,
// single columns, -1 where there is none (64 lanes hold the widest head).  Columns that are not
// turned are pairs of an angle of zero.
template <bool WIDE>
constexpr int kPairs = WIDE ? 4 : 2;
template <bool WIDE>
struct Columns {
    static constexpr int N = kPairs<WIDE>;
    int first[WIDE ? 1 : N], second[WIDE ? 1 : N];
    int unit[N];  // number of the pair, -1 where it is not turned
    bool live;
    __device__ void start(const RotationArgs& a, int lane) {
        if constexpr (WIDE) {
            live = lane * 8 < a.dim;
            const bool turned = lane * 4 < a.pairs;
            first[0] = turned && !a.interleaved ? 4 * lane : 8 * lane;
            second[0] = turned && !a.interleaved ? a.pairs + 4 * lane : 8 * lane + 4;
#pragma unroll
            for (int j = 0; j < N; ++j) unit[j] = turned ? 4 * lane + j : -1;
        } else {
            live = true;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int u = lane + 64 * j;
                unit[j] = u < a.pairs ? u : -1;
                first[j] = u < a.pairs ? (a.interleaved ? 2 * u : u) : 2 * u;  // (2 pairs + 2 (u - pairs))
                second[j] = u < a.pairs ? (a.interleaved ? 2 * u + 1 : u + a.pairs) : 2 * u + 1;
                if (first[j] >= a.dim) first[j] = -1;
                if (second[j] >= a.dim) second[j] = -1;
            }
        }
    }
    template <class T>
    __device__ void load(const T* p, const RotationArgs& a, float (&u)[N], float (&v)[N]) const {
        if constexpr (WIDE) {
            vec<T, 4> lo = {}, hi = {};
            if (live) {
                lo = *reinterpret_cast<const vec<T, 4>*>(p + first[0]);
                hi = *reinterpret_cast<const vec<T, 4>*>(p + second[0]);
            }
            const bool across = a.interleaved && unit[0] >= 0;
            u[0] = float(lo[0]);
            u[1] = float(across ? lo[2] : lo[1]);
            u[2] = float(across ? hi[0] : lo[2]);
            u[3] = float(across ? hi[2] : lo[3]);
            v[0] = float(across ? lo[1] : hi[0]);
            v[1] = float(across ? lo[3] : hi[1]);
            v[2] = float(across ? hi[1] : hi[2]);
            v[3] = float(hi[3]);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                u[j] = first[j] >= 0 ? float(p[first[j]]) : 0.f;
                v[j] = second[j] >= 0 ? float(p[second[j]]) : 0.f;
            }
        }
    }
    template <class T>
    __device__ void store(T* p, const RotationArgs& a, const float (&u)[N], const float (&v)[N]) const {
        if constexpr (WIDE) {
            if (!live) return;
            const bool across = a.interleaved && unit[0] >= 0;
            const vec<T, 4> lo = {T(u[0]), T(across ? v[0] : u[1]), T(across ? u[1] : u[2]), T(across ? v[1] : u[3])};
            const vec<T, 4> hi = {T(across ? u[2] : v[0]), T(across ? v[2] : v[1]), T(across ? u[3] : v[2]), T(v[3])};
            *reinterpret_cast<vec<T, 4>*>(p + first[0]) = lo;
            *reinterpret_cast<vec<T, 4>*>(p + second[0]) = hi;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (first[j] >= 0) p[first[j]] = T(u[j]);
                if (second[j] >= 0) p[second[j]] = T(v[j]);
            }
        }
    }
};

// What a workgroup keeps in LDS of its tokens: positions, cosines and sines, made once for
// all heads, and how far each token stands from a tensor's start.
struct Tokens {
    float cos[kTokens][kMaxDim / 2], sin[kTokens][kMaxDim / 2];
    int position[kTokens];
    int64_t x[2][kTokens], y[2][kTokens], dy[2][kTokens];
};
// Tokens first..first + count.  The turn is taken in double, whose fraction is right for
// every position, and the sine of the fraction as a float, moved on to first order by what that
// leaves of it (up to 2^-26 turns, 9e-8 of an angle: more than a sine's own rounding where it is
// small).
__device__ inline void start_tokens(const RotationArgs& a, Tokens& t, int64_t first, int count) {
    for (int i = threadIdx.x; i < count; i += 256) {
        const int64_t at = first + i, batch = at / a.tokens, token = at - batch * a.tokens;
        t.position[i] = a.positions ? a.positions[at] : int(token);
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const Side& s = a.side[side];
            t.x[side][i] = batch * s.x_batch + token * s.x_token;
            t.y[side][i] = batch * s.y_batch + token * s.y_token;
            t.dy[side][i] = batch * s.dy_batch + token * s.dy_token;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count * a.pairs; i += 256) {
        const int token = i / a.pairs, pair = i - token * a.pairs;
        const double turns = t.position[token] * a.rates[pair], fraction = turns - rint(turns);
        const float near = float(fraction), left = float(fraction - near) * 6.28318530717958647693f;
        float sine, cosine;
        sincospif(2.f * near, &sine, &cosine);
        t.sin[token][pair] = fmaf(left, cosine, sine);
        t.cos[token][pair] = fmaf(-left, sine, cosine);
    }
    __syncthreads();
}
// A lane's cosines and sines of a token.
template <bool WIDE>
__device__ inline void turn_of(const Tokens& t, int token, const Columns<WIDE>& columns, float (&c)[kPairs<WIDE>],
                               float (&s)[kPairs<WIDE>]) {
    if constexpr (WIDE) {
        typedef float Quad __attribute__((ext_vector_type(4)));
        Quad cos = {1, 1, 1, 1}, sin = {};
        if (columns.unit[0] >= 0) {
            cos = *reinterpret_cast<const Quad*>(&t.cos[token][columns.unit[0]]);
            sin = *reinterpret_cast<const Quad*>(&t.sin[token][columns.unit[0]]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            c[j] = cos[j];
            s[j] = sin[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < kPairs<WIDE>; ++j) {
            c[j] = columns.unit[j] >= 0 ? t.cos[token][columns.unit[j]] : 1.f;
            s[j] = columns.unit[j] >= 0 ? t.sin[token][columns.unit[j]] : 0.f;
        }
    }
}
// Calls body(token, head) for every head of the workgroup's tokens, a group of lanes each, in
// the order in which they stand in memory.
template <int LANES, class F>
__device__ __attribute__((always_inline)) inline void each_head(const Side& side, int tokens, F body) {
    constexpr int kGroups = 256 / LANES;
    const bool heads_first = side.x_head <= side.x_token;  // neighbours are a token's heads
    const int inner = heads_first ? side.heads : tokens, outer = heads_first ? tokens : side.heads;
    const int group = threadIdx.x / LANES;
    int o = group / inner, i = group - o * inner;
    const int step_o = kGroups / inner, step_i = kGroups - step_o * inner;
    while (o < outer) {
        body(heads_first ? o : i, heads_first ? i : o);
        o += step_o;
        i += step_i;
        if (i >= inner) {
            i -= inner;
            ++o;
        }
    }
}
// A side's weights in a lane's columns; ones where there are none.
template <class T, bool WIDE>
__device__ inline void weights_of(const RotationArgs& a, const Side& side, const Columns<WIDE>& columns, float (&u)[kPairs<WIDE>],
                                  float (&v)[kPairs<WIDE>]) {
    if (side.weight) columns.load(reinterpret_cast<const T*>(side.weight), a, u, v);
    else
#pragma unroll
        for (int j = 0; j < kPairs<WIDE>; ++j) u[j] = v[j] = 1;
}

// A workgroup takes a few tokens, a group of LANES lanes one head's vector after another.
// Bound: HBM (2 x 8192 tokens, 16 + 4 heads of 128, bf16: 168 MB in 38 us, 4.4 TB/s; the
// gradient's 252 MB in 61, 4.1 TB/s; a copy 5.1).  Neighbouring groups read neighbouring
// vectors: with a token each, and so a token's heads apart, they met on the same few
// channels of memory (54 and 69 us).
template <class T, int LANES, bool WIDE>
__global__ __launch_bounds__(256) void rotation_forward_k(RotationArgs a) {
    constexpr int N = kPairs<WIDE>;
    __shared__ __align__(16) Tokens t;
    const int64_t first = int64_t(blockIdx.x) * a.most;
    const int count = int(min(int64_t(a.most), a.count - first));
    start_tokens(a, t, first, count);
    Columns<WIDE> columns;
    columns.start(a, threadIdx.x % LANES);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const Side& side = a.side[k];
        if (!side.heads) continue;
        float wu[N], wv[N];
        weights_of<T>(a, side, columns, wu, wv);
        each_head<LANES>(side, count, [&](int token, int head) __attribute__((always_inline)) {
            float u[N] = {}, v[N] = {};
            if (t.position[token] >= 0) {  // (a place without a token, whose row is zeros, is not read)
                columns.load(reinterpret_cast<const T*>(side.x) + t.x[k][token] + head * side.x_head, a, u, v);
                float up = 1, c[N], s[N];
                if (a.norm) {
                    float square = 0;
#pragma unroll
                    for (int j = 0; j < N; ++j) square += u[j] * u[j] + v[j] * v[j];
                    up = 1.f / sqrtf(sum_group<LANES>(square) / a.dim + a.eps);
                }
                turn_of(t, token, columns, c, s);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float x = u[j] * up * wu[j], y = v[j] * up * wv[j];
                    u[j] = x * c[j] - y * s[j];
                    v[j] = x * s[j] + y * c[j];
                }
            }
            columns.store(reinterpret_cast<T*>(side.y) + t.y[k][token] + head * side.y_head, a, u, v);
        });
    }
}

// With n = x up, up = (mean x^2 + eps)^(-1/2) and g the gradient turned back: the
// weight's gradient is the sum of g n, and x's up (g w - n mean(g w n)).  Workgroups go
// through the tokens with a stride; their sums are joined in fixed order.
template <class T, int LANES, bool WIDE>
__global__ __launch_bounds__(256) void rotation_gradient_k(RotationArgs a) {
    constexpr int kGroups = 256 / LANES, N = kPairs<WIDE>;
    __shared__ __align__(16) Tokens t;
    __shared__ float sums[kGroups][LANES * 2 * N + 1];
    const int lane = threadIdx.x % LANES;
    Columns<WIDE> columns;
    columns.start(a, lane);
    float du[2][N] = {}, dv[2][N] = {};
    for (int64_t first = int64_t(blockIdx.x) * a.most; first < a.count; first += int64_t(gridDim.x) * a.most) {
        const int count = int(min(int64_t(a.most), a.count - first));
        __syncthreads();
        start_tokens(a, t, first, count);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const Side& side = a.side[k];
            if (!side.heads) continue;
            float wu[N], wv[N];
            weights_of<T>(a, side, columns, wu, wv);
            each_head<LANES>(side, count, [&](int token, int head) __attribute__((always_inline)) {
                float u[N] = {}, v[N] = {}, gu[N] = {}, gv[N] = {};
                if (t.position[token] >= 0) {
                    columns.load(reinterpret_cast<const T*>(side.x) + t.x[k][token] + head * side.x_head, a, u, v);
                    columns.load(reinterpret_cast<const T*>(side.dy) + t.dy[k][token] + head * side.dy_head, a, gu, gv);
                    float c[N], s[N], square = 0, dot = 0;
                    turn_of(t, token, columns, c, s);
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float back = gu[j] * c[j] + gv[j] * s[j];
                        gv[j] = gv[j] * c[j] - gu[j] * s[j];
                        gu[j] = back;
                        square += u[j] * u[j] + v[j] * v[j];
                    }
                    const float up = a.norm ? 1.f / sqrtf(sum_group<LANES>(square) / a.dim + a.eps) : 1.f;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        u[j] *= up;
                        v[j] *= up;
                        du[k][j] += gu[j] * u[j];
                        dv[k][j] += gv[j] * v[j];
                        gu[j] *= wu[j];
                        gv[j] *= wv[j];
                        dot += gu[j] * u[j] + gv[j] * v[j];
                    }
                    const float mean = a.norm ? sum_group<LANES>(dot) / a.dim : 0.f;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        gu[j] = up * (gu[j] - u[j] * mean);
                        gv[j] = up * (gv[j] - v[j] * mean);
                    }
                }
                columns.store(reinterpret_cast<T*>(side.y) + t.y[k][token] + head * side.y_head, a, gu, gv);
            });
        }
    }
    if (!a.part) return;
    for (int keys = 0; keys < 2; ++keys) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j) {
            sums[threadIdx.x / LANES][lane * 2 * N + j] = du[keys][j];
            sums[threadIdx.x / LANES][lane * 2 * N + N + j] = dv[keys][j];
        }
        __syncthreads();
        // (in the order of the lanes' places; rotation_weights_k undoes it)
        for (int i = threadIdx.x; i < LANES * 2 * N; i += 256) {
            float total = 0;
            for (int g = 0; g < kGroups; ++g) total += sums[g][i];
            a.part[(int64_t(blockIdx.x) * 2 + keys) * (LANES * 2 * N) + i] = total;
        }
    }
}

// The workgroups' sums in order: 16 places and 64 runs of workgroups a workgroup.
template <class T, int LANES, bool WIDE>
__global__ __launch_bounds__(1024) void rotation_weights_k(RotationArgs a, int blocks, T* dq_weight, T* dk_weight) {
    constexpr int N = kPairs<WIDE>;
    __shared__ float sums[64][17];
    const int keys = blockIdx.y, in = threadIdx.x & 15, run = threadIdx.x >> 4, place = blockIdx.x * 16 + in;
    const int per = (blocks + 63) / 64;
    float total = 0;
    for (int b = run * per; b < min(blocks, (run + 1) * per); ++b) total += a.part[(int64_t(b) * 2 + keys) * (LANES * 2 * N) + place];
    sums[run][in] = total;
    __syncthreads();
    T* to = keys ? dk_weight : dq_weight;
    if (run || !to) return;
    for (int r = 1; r < 64; ++r) total += sums[r][in];
    const int lane = place / (2 * N), j = place % N;
    const bool second = place & N;
    Columns<WIDE> columns;
    columns.start(a, lane);
    int column;
    if constexpr (WIDE) {
        if (!columns.live) return;
        if (a.interleaved && columns.unit[0] >= 0) column = columns.first[0] + 2 * j + second;
        else column = (second ? columns.second[0] : columns.first[0]) + j;
    } else {
        column = second ? columns.second[j] : columns.first[j];
        if (column < 0) return;
    }
    to[column] = T(total);
}

// ---- on the host ----------------------------------------------------------------------------
// Checks a tensor [batch][tokens][heads][dim]; whether its rows are read four values at a time.
bool check_view(const cpde_rotation_shape& s, const cpde_heads* h, int heads, bool output) {
    require(h, "null argument");
    if (!heads || !s.batch || !s.tokens) return true;
    require(h->data, "null tensor");
    require(h->batch >= 0 && h->token >= 0 && h->head >= 0, "negative stride");
    constexpr int64_t kFar = int64_t(1) << 40;
    require(h->batch <= kFar && h->token <= kFar && h->head <= kFar, "invalid stride");
    if (output) {
        std::pair<int64_t, int64_t> axes[] = {{h->batch, s.batch}, {h->token, s.tokens}, {h->head, heads}};
        std::sort(std::begin(axes), std::end(axes));
        int64_t extent = s.head_dim;
        for (const auto& [stride, count] : axes) {
            if (count == 1) continue;
            require(stride >= extent, "output elements overlap");
            extent = stride * (count - 1) + extent;
        }
    }
    const int64_t size = int64_t(type_bytes(s.dtype));
    const auto whole = [&](int64_t stride) { return stride * size % (4 * size) == 0; };
    return reinterpret_cast<uintptr_t>(h->data) % (4 * size) == 0 && whole(h->batch) && whole(h->token) && whole(h->head);
}
bool whole_weight(const cpde_rotation_shape& s, const void* w) {
    return reinterpret_cast<uintptr_t>(w) % (4 * type_bytes(s.dtype)) == 0;
}

RotationArgs arguments(const Rotation& p, const int32_t* positions) {
    const auto& s = p.shape;
    RotationArgs a{};
    a.rates = p.rates;
    a.positions = positions;
    a.count = int64_t(s.batch) * s.tokens;
    a.tokens = s.tokens;
    a.dim = s.head_dim;
    a.pairs = s.rotated / 2;
    a.interleaved = s.interleaved;
    a.norm = s.norm;
    a.eps = s.eps;
    a.side[0].heads = s.heads;
    a.side[1].heads = s.kv_heads;
    return a;
}
void set_side(Side& side, const cpde_heads* x, const cpde_heads* y, const cpde_heads* dy, const void* weight) {
    side.x = static_cast<const char*>(x->data);
    side.x_batch = x->batch;
    side.x_token = x->token;
    side.x_head = x->head;
    side.y = static_cast<char*>(y->data);
    side.y_batch = y->batch;
    side.y_token = y->token;
    side.y_head = y->head;
    if (dy) {
        side.dy = static_cast<const char*>(dy->data);
        side.dy_batch = dy->batch;
        side.dy_token = dy->token;
        side.dy_head = dy->head;
    }
    side.weight = static_cast<const char*>(weight);
}
// Whether the columns come in whole fours (and, where not turned or interleaved, eights).
bool whole_columns(const cpde_rotation_shape& s) {
    return s.head_dim % 8 == 0 && s.rotated % 8 == 0;
}
template <class F>
void with_lanes(const cpde_rotation_shape& s, bool wide_columns, F body) {
    const std::true_type yes{};
    if (!wide_columns) body(std::integral_constant<int, 64>{}, std::false_type{});
    else if (s.head_dim <= 32) body(std::integral_constant<int, 4>{}, yes);
    else if (s.head_dim <= 64) body(std::integral_constant<int, 8>{}, yes);
    else if (s.head_dim <= 128) body(std::integral_constant<int, 16>{}, yes);
    else body(std::integral_constant<int, 32>{}, yes);
}
// Tokens a workgroup takes at once: as many as leave `blocks` workgroups a unit (forward eight,
// gradient four; the other way round 41 and 66 us for 38 and 61), but as many as give each
// group of lanes a vector (4 x 729 tokens, 4 + 4 heads of 32, with the gradient: 31 us without).
void share_tokens(const Device& d, RotationArgs& a, int blocks, int lanes) {
    const int heads = std::max(a.side[0].heads, a.side[1].heads), groups = 256 / lanes;
    const int64_t most = std::max<int64_t>(a.count / (int64_t(blocks) * d.compute_units), (groups + heads - 1) / heads);
    a.most = int(std::max<int64_t>(1, std::min<int64_t>(kTokens, most)));
}
constexpr int kGradientBlocks = 8;  // of a unit, at most

}  // namespace
}  // namespace cpde

struct cpde_rotation_s : cpde::Rotation {};
using namespace cpde;

extern "C" {

int cpde_rotation_create(cpde_device* dev, const cpde_rotation_shape* shape, cpde_rotation** out) {
    return guarded([&] {
        require(dev && shape && out, "null argument");
        *out = nullptr;
        const cpde_rotation_shape s = *shape;
        check_dtype(s.dtype);
        require(s.batch >= 0 && s.tokens >= 0, "negative size");
        require(s.heads >= 0 && s.kv_heads >= 0 && s.heads + int64_t(s.kv_heads) >= 1 && s.heads + int64_t(s.kv_heads) <= 1 << 16,
                "1 to 65536 heads");
        require(s.head_dim >= 1 && s.head_dim <= kMaxDim, "a head is 1 to 256 wide");
        require(s.rotated >= 0 && s.rotated <= s.head_dim && s.rotated % 2 == 0, "an even number of a head's columns is rotated");
        require(s.base > 0 && std::isfinite(s.base), "the base is positive");
        require(s.eps >= 0 && std::isfinite(s.eps), "eps is not negative");
        require(int64_t(s.batch) * s.tokens <= int64_t(1) << 27, "too many tokens");
        require(!dev->capturing, "a capture is open on this device");
        OnDevice on(*dev);
        auto p = std::make_unique<cpde_rotation_s>();
        p->dev = dev;
        p->shape = s;
        p->blocks = dev->compute_units * kGradientBlocks;
        const size_t pairs = size_t(s.rotated / 2), part = s.backward ? size_t(p->blocks) * 2 * kMaxDim : 0;
        char* memory = nullptr;
        HIP_CHECK(hipMalloc(&memory, kMaxDim * sizeof(double) + part * sizeof(float)));
        p->rates = reinterpret_cast<double*>(memory);
        p->part = part ? reinterpret_cast<float*>(memory + kMaxDim * sizeof(double)) : nullptr;
        std::vector<double> rates(pairs);
        for (size_t i = 0; i < pairs; ++i)
            rates[i] = std::pow(double(s.base), -2.0 * double(i) / s.rotated) / 6.283185307179586476925;
        const hipError_t copied = pairs ? hipMemcpy(p->rates, rates.data(), pairs * sizeof(double), hipMemcpyHostToDevice) : hipSuccess;
        if (copied != hipSuccess) (void)hipFree(memory);
        HIP_CHECK(copied);
        *out = p.release();
    });
}

int cpde_rotation_destroy(cpde_rotation* rotation) {
    return guarded([&] {
        if (!rotation) return;
        OnDevice on(*rotation->dev);
        sync_stream(*rotation->dev, __LINE__);
        ++rotation->dev->layout;
        HIP_CHECK(hipFree(rotation->rates));
        delete rotation;
    });
}

int cpde_rotation_forward(cpde_rotation* rotation, const cpde_heads* q, const cpde_heads* k, const void* q_weight,
                          const void* k_weight, const int32_t* positions, const cpde_heads* q_out,
                          const cpde_heads* k_out) {
    return guarded([&] {
        require(rotation, "null argument");
        const Rotation& p = *rotation;
        const auto& s = p.shape;
        RotationArgs a = arguments(p, positions);
        bool whole = whole_columns(s) && whole_weight(s, q_weight) && whole_weight(s, k_weight);
        if (s.heads) {
            whole = check_view(s, q, s.heads, false) && whole;
            whole = check_view(s, q_out, s.heads, true) && whole;
            set_side(a.side[0], q, q_out, nullptr, q_weight);
        }
        if (s.kv_heads) {
            whole = check_view(s, k, s.kv_heads, false) && whole;
            whole = check_view(s, k_out, s.kv_heads, true) && whole;
            set_side(a.side[1], k, k_out, nullptr, k_weight);
        }
        if (!a.count) return;
        Device& d = *p.dev;
        OnDevice on(d);
        flush_reduce(d);
        TraceScope trace(d, kTraceRotation, 2.0 * a.count * (s.heads + s.kv_heads) * s.head_dim * type_bytes(s.dtype));
        with_type(s.dtype, [&](auto element) {
            using T = decltype(element);
            with_lanes(s, whole, [&](auto lanes, auto whole_) {
                constexpr int L = decltype(lanes)::value;
                share_tokens(d, a, 8, L);
                const int64_t blocks = (a.count + a.most - 1) / a.most;
                hipLaunchKernelGGL((rotation_forward_k<T, L, decltype(whole_)::value>), unsigned(blocks), 256, 0, d.stream, a);
            });
        });
        HIP_CHECK(hipGetLastError());
    });
}

int cpde_rotation_backward(cpde_rotation* rotation, const cpde_heads* q, const cpde_heads* k, const void* q_weight,
                           const void* k_weight, const int32_t* positions, const cpde_heads* dq_out,
                           const cpde_heads* dk_out, const cpde_heads* dq, const cpde_heads* dk, void* dq_weight,
                           void* dk_weight) {
    return guarded([&] {
        require(rotation, "null argument");
        const Rotation& p = *rotation;
        const auto& s = p.shape;
        require(s.backward, "the plan was created without a backward");
        RotationArgs a = arguments(p, positions);
        bool whole = whole_columns(s) && whole_weight(s, q_weight) && whole_weight(s, k_weight);
        if (s.heads) {
            whole = check_view(s, q, s.heads, false) && whole;
            whole = check_view(s, dq_out, s.heads, false) && whole;
            whole = check_view(s, dq, s.heads, true) && whole;
            set_side(a.side[0], q, dq, dq_out, q_weight);
        }
        if (s.kv_heads) {
            whole = check_view(s, k, s.kv_heads, false) && whole;
            whole = check_view(s, dk_out, s.kv_heads, false) && whole;
            whole = check_view(s, dk, s.kv_heads, true) && whole;
            set_side(a.side[1], k, dk, dk_out, k_weight);
        }
        if (!s.kv_heads) dk_weight = nullptr;
        if (!s.heads) dq_weight = nullptr;
        if (dq_weight || dk_weight) a.part = p.part;
        else if (!a.count) return;
        Device& d = *p.dev;
        OnDevice on(d);
        flush_reduce(d);
        TraceScope trace(d, kTraceRotation, 3.0 * a.count * (s.heads + s.kv_heads) * s.head_dim * type_bytes(s.dtype));
        with_type(s.dtype, [&](auto element) {
            using T = decltype(element);
            with_lanes(s, whole, [&](auto lanes, auto whole_) {
                constexpr int L = decltype(lanes)::value;
                constexpr bool W = decltype(whole_)::value;
                share_tokens(d, a, 4, L);
                const int64_t want = (a.count + a.most - 1) / a.most;
                const int blocks = int(std::max<int64_t>(1, std::min<int64_t>(want, p.blocks)));
                hipLaunchKernelGGL((rotation_gradient_k<T, L, W>), blocks, 256, 0, d.stream, a);
                HIP_CHECK(hipGetLastError());
                if (a.part)
                    hipLaunchKernelGGL((rotation_weights_k<T, L, W>), dim3(L * 2 * kPairs<W> / 16, 2), 1024, 0, d.stream, a, blocks,
                                       static_cast<T*>(dq_weight), static_cast<T*>(dk_weight));
            });
        });
        HIP_CHECK(hipGetLastError());
    });
}

}  // extern "C"
