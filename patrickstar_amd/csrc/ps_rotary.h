// Kernels of ps_rotate_heads and ps_norm_rotate_heads_backward.
//
// A workgroup has either queries or keys.  A wave's lanes are cut into groups of G (a power of two); a group takes one head of one
// token at a time.  A lane holds one vector of first members of pairs and the vector of their partners ("unit"), so a rotation
// needs no other lane, and the norm only a sum over the group.  Turning angles depend on token and pair alone: the lanes of a wave
// make each of its tokens' cosines and sines once, one pair a lane, and hand them round in LDS.
//
// All of it is bound by memory: 6 to 17 operations for every element that is read and written.  Measured (bf16, GPU time):
//   rotation, 12000 tokens x 32 heads x 128            31 us, 197 MB, 6.3 TB/s
//   norm and rotation, 16383 x 40 x 128                57 us, 335 MB, 5.9 TB/s
//   its gradient                                      105 us, 503 MB, 4.8 TB/s (three streams; a copy of rows on this GPU 4.8 to 5.2)
//   fp16, 16384 x 50 x 64 with neighbouring pairs      33 us, 210 MB, 6.3 TB/s
// What it takes: 8 bytes a lane of 16-bit types, not 16, for twice the waves (gradient 131 us with 16); queries and keys apart, so
// that a lane holds one weight and one sum (gradient 315 us with both); angles once a token, not once a group (with the former
// 315 -> 148); the next head on its way while this one is worked on; stores past the caches where the outputs are longer than they
// are (rotation 39 us without, the gradient 119), which needs whole lines: with neighbouring pairs a unit is one access of 16 bytes
// (44 us with two).
#ifndef PS_ROTARY_H
#define PS_ROTARY_H

#include "ps_vec.h"

namespace {

constexpr int kHeadsBlock = 256, kHeadsWaves = kHeadsBlock / 64;

// The workgroups of queries, or of keys.
struct HeadsPart {
    const void* x;
    const void* grad;
    void* out;
    const void* weight;
    float* partial;      // workgroups x dim: sums of the weights' gradient
    int64_t x_stride[3];
    int64_t grad_stride[3];
    uint32_t items;      // (tokens of a wave) x (splits of a token's heads)
    uint32_t blocks;
    int heads;
    int slot_shift;      // log2 of the groups that share a token
    int split_shift;     // log2 of the waves that share a token
    bool weight_vectors; // the weight is aligned like a vector of its type
};

struct HeadsArgs {
    HeadsPart part[2];
    const void* positions;
    const int64_t* plan;
    int64_t position_stride[3];
    uint32_t tokens, all_tokens;  // of a batch's row, of the call
    int dim, pairs;
    int group_shift;  // log2 of G
    float eps, inv_dim;
    bool one_axis;    // the position need not wait for the plan
    bool weight_f32, positions_64, interleaved, inverse;
    bool whole;       // every unit's two vectors are one, aligned as such
};

// cos and sin of `phase` / 2^32 turns.  The instructions take turns; over all of [-1/2, 1/2) in steps of 2^-24 their largest error is
// 1.3e-7, as good as a polynomial of a dozen instructions.
__device__ __forceinline__ void cos_sin(int32_t phase, float& c, float& s)
{
    const float x = (float)phase * 0x1p-32f;
    c = __builtin_amdgcn_cosf(x);
    s = __builtin_amdgcn_sinf(x);
}

// Sum over the lanes of a group; every lane gets it.  Within 16 lanes by moves between lanes as part of the addition, which take
// no LDS.
__device__ __forceinline__ float group_sum(float v, int group_shift)
{
    if (group_shift > 0) v += moved<0xB1>(v);   // the other of a pair
    if (group_shift > 1) v += moved<0x4E>(v);   // the other pair of four
    if (group_shift > 2) v += moved<0x141>(v);  // mirrored in eight: fours are alike by now
    if (group_shift > 3) v += moved<0x140>(v);  // mirrored in sixteen
    if (group_shift > 4) v += __shfl_xor(v, 16);
    if (group_shift > 5) v += __shfl_xor(v, 32);
    return v;
}

// Where a unit's two vectors lie (in elements), and which pairs they are.
struct Unit {
    int a, b;      // b < 0: there is no second one
    int pair;      // first pair; < 0: not rotated
    bool there;
    bool alternate;  // members and partners alternate in memory
};

template <int V>
__device__ __forceinline__ Unit unit_of(const HeadsArgs& p, int u)
{
    Unit r;
    const int turned = p.pairs / V;  // units
    r.there = 2 * V * u < p.dim;
    if (p.interleaved || u >= turned) {
        r.a = 2 * V * u;
        r.b = r.a + V < p.dim ? r.a + V : -1;
    } else {
        r.a = V * u;
        r.b = r.a + p.pairs;
    }
    r.pair = u < turned ? V * u : -1;
    r.alternate = V > 1 && p.interleaved && r.pair >= 0;
    return r;
}

template <int V>
struct Halves {
    float a[V], b[V];
};

// A unit as it lies in memory.
template <typename T, int V>
struct Raw {
    typename VecOf<T, V>::type a, b;

    // `whole`: the two are one vector of 2 V elements
    __device__ __forceinline__ void load(const T* row, const Unit& u, bool whole)
    {
        if (whole) {
            const auto both = load_raw<T, 2 * V>(row + u.a);
#pragma unroll
            for (int e = 0; e < V; ++e) put<T, V>(a, e, both[e]), put<T, V>(b, e, both[V + e]);
            return;
        }
        a = load_raw<T, V>(row + u.a);
        b = u.b >= 0 ? load_raw<T, V>(row + u.b) : typename VecOf<T, V>::type{};
    }
    template <bool STREAM>
    __device__ __forceinline__ void store(T* row, const Unit& u, bool whole) const
    {
        if (whole) {
            typename VecOf<T, 2 * V>::type both;
#pragma unroll
            for (int e = 0; e < V; ++e) both[e] = get<T, V>(a, e), both[V + e] = get<T, V>(b, e);
            store_raw<T, 2 * V, STREAM>(row + u.a, both);
            return;
        }
        store_raw<T, V, STREAM>(row + u.a, a);
        if (u.b >= 0) store_raw<T, V, STREAM>(row + u.b, b);
    }
    __device__ __forceinline__ Halves<V> halves(const Unit& u) const
    {
        Halves<V> r;
#pragma unroll
        for (int e = 0; e < V; ++e) r.a[e] = element<T, V>(a, e), r.b[e] = element<T, V>(b, e);
        if (V > 1 && u.alternate) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                r.a[e] = 2 * e < V ? element<T, V>(a, 2 * e) : element<T, V>(b, 2 * e - V);
                r.b[e] = 2 * e + 1 < V ? element<T, V>(a, 2 * e + 1) : element<T, V>(b, 2 * e + 1 - V);
            }
        }
        return r;
    }
    __device__ __forceinline__ void set(const Halves<V>& h, const Unit& u)
    {
        if (V > 1 && u.alternate) {
            float x[2 * V];
#pragma unroll
            for (int e = 0; e < V; ++e) x[2 * e] = h.a[e], x[2 * e + 1] = h.b[e];
#pragma unroll
            for (int e = 0; e < V; ++e) set_element<T, V>(a, e, x[e]), set_element<T, V>(b, e, x[V + e]);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) set_element<T, V>(a, e, h.a[e]), set_element<T, V>(b, e, h.b[e]);
        }
    }
};

template <typename T, int V>
__device__ __forceinline__ Halves<V> weight_of(const void* weight, bool vectors, const Unit& u)
{
    const T* w = static_cast<const T*>(weight);
    Raw<T, V> r;
    if (vectors) {
        r.load(w, u, false);
    } else {
        r.b = typename VecOf<T, V>::type{};
#pragma unroll
        for (int e = 0; e < V; ++e) {
            put<T, V>(r.a, e, global(w)[u.a + e]);
            if (u.b >= 0) put<T, V>(r.b, e, global(w)[u.b + e]);
        }
    }
    return r.halves(u);
}

template <typename T, int V>
__device__ __forceinline__ Halves<V> load_weight(const HeadsArgs& p, const HeadsPart& part, const Unit& u)
{
    if (part.weight == nullptr) {
        Halves<V> w;
#pragma unroll
        for (int e = 0; e < V; ++e) w.a[e] = w.b[e] = 1.0f;
        return w;
    }
    // (fp32 weights of a vector of 8 are two vectors each: left to the compiler, element by element)
    if (p.weight_f32) return weight_of<float, V>(part.weight, part.weight_vectors && V <= 4, u);
    return weight_of<T, V>(part.weight, part.weight_vectors, u);
}

// What a wave does in one turn of its loop: a group of tokens, and a part of their heads.
struct Item {
    uint32_t first_token, token;  // of the wave, of the lane's group
    int64_t b, t;
    int slot;                     // the lane's token among the wave's
    int head, step;
    bool there;
};

__device__ __forceinline__ Item item_of(const HeadsArgs& p, const HeadsPart& part, uint32_t number)
{
    const int group = (threadIdx.x & 63) >> p.group_shift;
    const int tokens_shift = 6 - p.group_shift - part.slot_shift;
    Item r;
    r.first_token = (number >> part.split_shift) << tokens_shift;
    r.slot = group >> part.slot_shift;
    r.token = r.first_token + (uint32_t)r.slot;
    r.there = r.token < p.all_tokens;
    const uint32_t token = r.there ? r.token : 0;
    r.b = token / p.tokens;
    r.t = token % p.tokens;
    r.head = (group & ((1 << part.slot_shift) - 1)) + (int)((number & ((1u << part.split_shift) - 1)) << part.slot_shift);
    r.step = 1 << (part.slot_shift + part.split_shift);
    return r;
}

// Pairs of a wave's tokens: at most (64 / G groups) x (G lanes x U units x V pairs).
template <int V, int U>
constexpr int kTurns = 64 * U * V;

// The lanes' cosines and sines of a wave's tokens, made one pair a lane and handed round in the wave's own LDS.
template <int V, int U>
__device__ __forceinline__ void make_turns(const HeadsArgs& p, const HeadsPart& part, const Item& item, const Unit (&units)[U], float2* lds,
                                           float (&c)[U][V], float (&s)[U][V])
{
    const int tokens_shift = 6 - p.group_shift - part.slot_shift;
    const int lane = threadIdx.x & 63, all = p.pairs << tokens_shift;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the last turn's reads are done
    __builtin_amdgcn_wave_barrier();
    for (int i = lane; i < all; i += 64) {
        const uint32_t slot = (uint32_t)i / (uint32_t)p.pairs, pair = (uint32_t)i % (uint32_t)p.pairs;
        const uint32_t token = item.first_token + slot;
        if (token >= p.all_tokens) break;
        const int64_t step = global(p.plan)[2 * pair], axis = p.one_axis ? 0 : global(p.plan)[2 * pair + 1];
        const int64_t at = axis * p.position_stride[0] + (token / p.tokens) * p.position_stride[1] + (token % p.tokens) * p.position_stride[2];
        const int64_t position = p.positions_64 ? global(static_cast<const int64_t*>(p.positions))[at]
                                                : global(static_cast<const int32_t*>(p.positions))[at];
        float2 turn;
        cos_sin((int32_t)(((uint64_t)position * (uint64_t)step) >> 32), turn.x, turn.y);
        if (p.inverse) turn.y = -turn.y;
        lds[i] = turn;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const bool turned = units[k].there && units[k].pair >= 0;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float2 turn = turned ? lds[item.slot * p.pairs + units[k].pair + e] : make_float2(1.0f, 0.0f);
            c[k][e] = turn.x;
            s[k][e] = turn.y;
        }
    }
}

template <int V>
__device__ __forceinline__ void turn(Halves<V>& x, const float (&c)[V], const float (&s)[V])
{
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float a = x.a[e], b = x.b[e];
        x.a[e] = __builtin_fmaf(a, c[e], -(b * s[e]));
        x.b[e] = __builtin_fmaf(b, c[e], a * s[e]);
    }
}

// Forward, and backward of a rotation alone (the other way round).  One pass: a head's elements are read once, and its norm is a sum of
// squares over the lanes that hold them.
template <typename T, int V, int U, bool NORM, bool STREAM>
__global__ __launch_bounds__(kHeadsBlock) void rotate_heads_kernel(HeadsArgs p)
{
    __shared__ float2 turns[kHeadsWaves][kTurns<V, U>];
    const bool keys = blockIdx.x >= p.part[0].blocks;
    const HeadsPart& part = p.part[keys];
    const uint32_t block = blockIdx.x - (keys ? p.part[0].blocks : 0);
    const int wave = threadIdx.x >> 6;
    Unit units[U];
    Halves<V> w[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
        units[k] = unit_of<V>(p, (threadIdx.x & ((1 << p.group_shift) - 1)) + (k << p.group_shift));
        if (NORM && units[k].there) w[k] = load_weight<T, V>(p, part, units[k]);
    }
    for (uint32_t number = block * kHeadsWaves + wave; number < part.items; number += part.blocks * kHeadsWaves) {
        const Item item = item_of(p, part, number);
        const T* x = static_cast<const T*>(part.x) + item.b * part.x_stride[0] + item.t * part.x_stride[1];
        T* out = static_cast<T*>(part.out) + (int64_t)item.token * part.heads * p.dim;
        const int heads = item.there ? part.heads : 0;
        int head = item.head;
        // the first head is on its way while the angles are made
        Raw<T, V> next[U];
        if (head < heads) {
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (units[k].there) next[k].load(x + head * part.x_stride[2], units[k], p.whole);
        }
        float c[U][V], s[U][V];
        make_turns<V, U>(p, part, item, units, turns[wave], c, s);
        for (; head < heads; head += item.step) {
            Halves<V> v[U];
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (!units[k].there) continue;
                v[k] = next[k].halves(units[k]);
                if (NORM) {
#pragma unroll
                    for (int e = 0; e < V; ++e) sum = __builtin_fmaf(v[k].a[e], v[k].a[e], __builtin_fmaf(v[k].b[e], v[k].b[e], sum));
                }
            }
            if (head + item.step < heads) {
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (units[k].there) next[k].load(x + (head + item.step) * part.x_stride[2], units[k], p.whole);
            }
            if (NORM) {
                const float r = __builtin_amdgcn_rsqf(__builtin_fmaf(group_sum(sum, p.group_shift), p.inv_dim, p.eps));
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    if (!units[k].there) continue;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        v[k].a[e] = v[k].a[e] * r * w[k].a[e];
                        v[k].b[e] = v[k].b[e] * r * w[k].b[e];
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (!units[k].there) continue;
                turn<V>(v[k], c[k], s[k]);
                Raw<T, V> result;
                result.set(v[k], units[k]);
                result.template store<STREAM>(out + (int64_t)head * p.dim, units[k], p.whole);
            }
        }
    }
}

// With dy the gradient turned back, r = 1 / rms(x) and y = x r w:
//   dw = sum over tokens and heads of dy x r,   dx = r (w dy - x r^2 mean(x w dy)).
// The root is made again from x, which has to be read anyway.  A lane keeps its part of dw in registers over all heads and tokens
// that it takes; a workgroup leaves one row of sums, and sum_weight_grads_kernel adds the rows in their order: no atomics.
template <typename T, int V, int U, bool STREAM>
__global__ __launch_bounds__(kHeadsBlock) void norm_rotate_heads_backward_kernel(HeadsArgs p)
{
    __shared__ float2 turns[kHeadsWaves][kTurns<V, U>];
    __shared__ float sums[PS_MAX_HEAD_DIM];
    const bool keys = blockIdx.x >= p.part[0].blocks;
    const HeadsPart& part = p.part[keys];
    const uint32_t block = blockIdx.x - (keys ? p.part[0].blocks : 0);
    const int wave = threadIdx.x >> 6;
    Unit units[U];
    Halves<V> w[U], dw[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
        units[k] = unit_of<V>(p, (threadIdx.x & ((1 << p.group_shift) - 1)) + (k << p.group_shift));
        if (units[k].there) w[k] = load_weight<T, V>(p, part, units[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[k].a[e] = dw[k].b[e] = 0.0f;
    }
    for (uint32_t number = block * kHeadsWaves + wave; number < part.items; number += part.blocks * kHeadsWaves) {
        const Item item = item_of(p, part, number);
        const T* x = static_cast<const T*>(part.x) + item.b * part.x_stride[0] + item.t * part.x_stride[1];
        const T* g = static_cast<const T*>(part.grad) + item.b * part.grad_stride[0] + item.t * part.grad_stride[1];
        T* out = static_cast<T*>(part.out) + (int64_t)item.token * part.heads * p.dim;
        const int heads = item.there ? part.heads : 0;
        int head = item.head;
        Raw<T, V> next_x[U], next_g[U];
        if (head < heads) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (!units[k].there) continue;
                next_x[k].load(x + head * part.x_stride[2], units[k], p.whole);
                next_g[k].load(g + head * part.grad_stride[2], units[k], p.whole);
            }
        }
        float c[U][V], s[U][V];
        make_turns<V, U>(p, part, item, units, turns[wave], c, s);
#pragma unroll 1
        for (; head < heads; head += item.step) {
            Halves<V> v[U], d[U];
            float square = 0.0f, dot = 0.0f;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (!units[k].there) continue;
                v[k] = next_x[k].halves(units[k]);
                d[k] = next_g[k].halves(units[k]);
            }
            if (head + item.step < heads) {
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    if (!units[k].there) continue;
                    next_x[k].load(x + (head + item.step) * part.x_stride[2], units[k], p.whole);
                    next_g[k].load(g + (head + item.step) * part.grad_stride[2], units[k], p.whole);
                }
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (!units[k].there) continue;
                turn<V>(d[k], c[k], s[k]);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    square = __builtin_fmaf(v[k].a[e], v[k].a[e], __builtin_fmaf(v[k].b[e], v[k].b[e], square));
                    dot = __builtin_fmaf(v[k].a[e] * w[k].a[e], d[k].a[e], __builtin_fmaf(v[k].b[e] * w[k].b[e], d[k].b[e], dot));
                }
            }
            square = group_sum(square, p.group_shift);
            dot = group_sum(dot, p.group_shift);
            const float r = __builtin_amdgcn_rsqf(__builtin_fmaf(square, p.inv_dim, p.eps));
            const float back = r * r * (dot * p.inv_dim);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (!units[k].there) continue;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float da = d[k].a[e], db = d[k].b[e];
                    dw[k].a[e] = __builtin_fmaf(da, v[k].a[e] * r, dw[k].a[e]);
                    dw[k].b[e] = __builtin_fmaf(db, v[k].b[e] * r, dw[k].b[e]);
                    d[k].a[e] = r * __builtin_fmaf(-v[k].a[e], back, w[k].a[e] * da);
                    d[k].b[e] = r * __builtin_fmaf(-v[k].b[e], back, w[k].b[e] * db);
                }
                Raw<T, V> result;
                result.set(d[k], units[k]);
                result.template store<STREAM>(out + (int64_t)head * p.dim, units[k], p.whole);
            }
        }
    }
    if (part.partial == nullptr) return;
    // groups of a wave, then the waves one after another
    for (int i = threadIdx.x; i < p.dim; i += kHeadsBlock) sums[i] = 0.0f;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e)
            for (int m = 1 << p.group_shift; m < 64; m <<= 1) {
                dw[k].a[e] += __shfl_xor(dw[k].a[e], m);
                dw[k].b[e] += __shfl_xor(dw[k].b[e], m);
            }
    for (int turn = 0; turn < kHeadsWaves; ++turn) {
        if (turn == wave && (threadIdx.x & 63) < (1u << p.group_shift)) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (!units[k].there) continue;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    sums[units[k].alternate ? units[k].a + 2 * e : units[k].a + e] += dw[k].a[e];
                    if (units[k].b >= 0) sums[units[k].alternate ? units[k].a + 2 * e + 1 : units[k].b + e] += dw[k].b[e];
                }
            }
        }
        __syncthreads();
    }
    float* row = part.partial + (int64_t)block * p.dim;
    for (int i = threadIdx.x; i < p.dim; i += kHeadsBlock) global(row)[i] = sums[i];
}

// Columns over workgroups, rows over a workgroup's slices in a fixed order: 1024 rows of 128 columns take 4 us, which is their
// reads' latency (13 with a slice's reads one after another).
constexpr int kSumColumns = 16, kSumSlices = 64;

struct WeightGrads {
    const float* partial[2];  // rows x dim
    void* out[2];
    int rows[2];
    int dim;
    bool f32;
};

// blockIdx.y: of the queries' weight, of the keys'.
template <typename T>
__global__ __launch_bounds__(kSumColumns * kSumSlices) void sum_weight_grads_kernel(WeightGrads p)
{
    __shared__ float sums[kSumSlices][kSumColumns + 1];
    const int which = blockIdx.y, column = threadIdx.x % kSumColumns, slice = threadIdx.x / kSumColumns;
    const int at = blockIdx.x * kSumColumns + column;
    if (p.out[which] == nullptr) return;
    float sum = 0.0f;
    if (at < p.dim)
        for (int r = slice; r < p.rows[which]; r += 4 * kSumSlices) {
            float part[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int row = r + k * kSumSlices;
                part[k] = row < p.rows[which] ? global(p.partial[which])[(int64_t)row * p.dim + at] : 0.0f;
            }
            sum += (part[0] + part[1]) + (part[2] + part[3]);
        }
    sums[slice][column] = sum;
    __syncthreads();
    if (slice != 0 || at >= p.dim) return;
    sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kSumSlices; ++k) sum += sums[k][column];
    if (p.f32)
        global(static_cast<float*>(p.out[which]))[at] = sum;
    else
        global(static_cast<T*>(p.out[which]))[at] = from_float<T>(sum);
}

}  // namespace

#endif  // PS_ROTARY_H
