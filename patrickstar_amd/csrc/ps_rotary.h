// Kernels of ps_rotate_heads and ps_norm_rotate_heads_backward.
//
// A wave's lanes are cut into groups of G (a power of two); a group takes one head of one token at a time.  A lane holds one
// vector of first members of pairs and the vector of their partners ("unit"), so a rotation needs no other lane, and the norm only
// a sum over the group.  Turning angles depend on token and pair alone: a lane makes its V cosines and sines once and keeps them
// for every head of the token that its group takes.
#ifndef PS_ROTARY_H
#define PS_ROTARY_H

#include "ps_vec.h"

namespace {

struct HeadsArgs {
    const void* x[2];
    const void* grad[2];
    void* out[2];
    const void* weight[2];
    const void* positions;
    const int64_t* plan;
    int64_t x_stride[2][3];
    int64_t grad_stride[2][3];
    int64_t position_stride[3];
    uint32_t tokens, all_tokens;  // of a batch's row, of the call
    int heads[2];
    int dim, pairs;
    int group_shift;  // log2 of G
    int slot_shift;   // log2 of the groups that share a token
    float eps, inv_dim;
    float* partial;   // workgroups x 2 x dim: sums of the weights' gradients
    bool weight_f32, positions_64, interleaved, inverse;
};

// cos and sin of `phase` / 2^32 turns.  Whole quarters come off exactly; what is left lies in [-pi/4, pi/4], where the Taylor
// polynomials to x^9 and x^10 are within 2e-9 of the functions.
__device__ __forceinline__ void cos_sin(int32_t phase, float& c, float& s)
{
    const int32_t quarter = (int32_t)(((uint32_t)phase + 0x20000000u) >> 30);
    const int32_t rest = (int32_t)((uint32_t)phase - ((uint32_t)quarter << 30));
    const float x = (float)rest * 1.4629180792671596e-9f;  // 2 pi / 2^32
    const float x2 = x * x;
    float ps = 2.7557319e-6f;
    ps = __builtin_fmaf(ps, x2, -1.9841270e-4f);
    ps = __builtin_fmaf(ps, x2, 8.3333333e-3f);
    ps = __builtin_fmaf(ps, x2, -1.6666667e-1f);
    const float sx = __builtin_fmaf(ps * x2, x, x);
    float pc = -2.7557319e-7f;
    pc = __builtin_fmaf(pc, x2, 2.4801587e-5f);
    pc = __builtin_fmaf(pc, x2, -1.3888889e-3f);
    pc = __builtin_fmaf(pc, x2, 4.1666667e-2f);
    pc = __builtin_fmaf(pc, x2, -0.5f);
    const float cx = __builtin_fmaf(pc, x2, 1.0f);
    const bool swap = quarter & 1;
    c = swap ? sx : cx;
    s = swap ? cx : sx;
    if (quarter == 1 || quarter == 2) c = -c;
    if (quarter & 2) s = -s;
}

__device__ __forceinline__ float group_sum(float v, int group_shift)
{
    for (int k = 0; k < group_shift; ++k) v += __shfl_xor(v, 1 << k);
    return v;
}

// Where a unit's two vectors lie, and which pairs they are: vectors a and b (in elements), or one of 2 V elements at a.
struct Unit {
    int a, b;      // first elements; b < 0: there is none
    int pair;      // first pair; < 0: not rotated
    bool there;
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
    return r;
}

template <typename T, int V>
struct Halves {
    float a[V], b[V];
};

template <typename T, int V>
__device__ __forceinline__ Halves<T, V> load_unit(const T* row, const Unit& u, bool interleaved)
{
    Halves<T, V> r;
    load_vec<T, V>(row + u.a, r.a);
    if (u.b >= 0) {
        load_vec<T, V>(row + u.b, r.b);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) r.b[e] = 0.0f;
    }
    if (V > 1 && interleaved && u.pair >= 0) {  // members and partners alternate
        Halves<T, V> t = r;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            r.a[e] = 2 * e < V ? t.a[2 * e] : t.b[2 * e - V];
            r.b[e] = 2 * e + 1 < V ? t.a[2 * e + 1] : t.b[2 * e + 1 - V];
        }
    }
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_unit(T* row, const Unit& u, bool interleaved, const Halves<T, V>& v)
{
    Halves<T, V> t = v;
    if (V > 1 && interleaved && u.pair >= 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (2 * e < V)
                t.a[2 * e] = v.a[e];
            else
                t.b[2 * e - V] = v.a[e];
            if (2 * e + 1 < V)
                t.a[2 * e + 1] = v.b[e];
            else
                t.b[2 * e + 1 - V] = v.b[e];
        }
    }
    store_vec<T, V>(row + u.a, t.a);
    if (u.b >= 0) store_vec<T, V>(row + u.b, t.b);
}

template <typename T, int V>
__device__ __forceinline__ Halves<T, V> load_weight(const HeadsArgs& p, int which, const Unit& u)
{
    Halves<T, V> w;
    if (p.weight[which] == nullptr) {
#pragma unroll
        for (int e = 0; e < V; ++e) w.a[e] = w.b[e] = 1.0f;
        return w;
    }
    if (p.weight_f32) {  // element by element: its address need not be a vector's
        const float* f = static_cast<const float*>(p.weight[which]);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const bool alternate = p.interleaved && u.pair >= 0;
            const int a = alternate ? u.a + 2 * e : u.a + e, b = alternate ? u.a + 2 * e + 1 : u.b + e;
            w.a[e] = global(f)[a];
            w.b[e] = u.b >= 0 ? global(f)[b] : 0.0f;
        }
        return w;
    }
    const T* f = static_cast<const T*>(p.weight[which]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const bool alternate = p.interleaved && u.pair >= 0;
        const int a = alternate ? u.a + 2 * e : u.a + e, b = alternate ? u.a + 2 * e + 1 : u.b + e;
        w.a[e] = to_float<T>(global(f)[a]);
        w.b[e] = u.b >= 0 ? to_float<T>(global(f)[b]) : 0.0f;
    }
    return w;
}

template <int V, int U>
__device__ __forceinline__ void make_turns(const HeadsArgs& p, const Unit (&units)[U], int64_t position_at, float (&c)[U][V],
                                           float (&s)[U][V])
{
#pragma unroll
    for (int k = 0; k < U; ++k) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            c[k][e] = 1.0f;
            s[k][e] = 0.0f;
            if (units[k].there && units[k].pair >= 0) {
                const int64_t step = global(p.plan)[2 * (units[k].pair + e)];
                const int64_t at = position_at + global(p.plan)[2 * (units[k].pair + e) + 1] * p.position_stride[0];
                const int64_t position = p.positions_64 ? global(static_cast<const int64_t*>(p.positions))[at]
                                                        : global(static_cast<const int32_t*>(p.positions))[at];
                cos_sin((int32_t)(((uint64_t)position * (uint64_t)step) >> 32), c[k][e], s[k][e]);
                if (p.inverse) s[k][e] = -s[k][e];
            }
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void turn(Halves<T, V>& x, const float (&c)[V], const float (&s)[V])
{
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float a = x.a[e], b = x.b[e];
        x.a[e] = __builtin_fmaf(a, c[e], -(b * s[e]));
        x.b[e] = __builtin_fmaf(b, c[e], a * s[e]);
    }
}

// The wave's part of a call: which token a lane's group has, and where its heads begin.
struct Slot {
    uint32_t token;
    int head;  // of queries and keys together
    int lane_in_group;
    bool there;
};

__device__ __forceinline__ Slot slot_of(const HeadsArgs& p, uint32_t wave)
{
    const int lane = threadIdx.x & 63;
    const int group = lane >> p.group_shift;
    const int tokens_shift = 6 - p.group_shift - p.slot_shift;
    Slot r;
    r.token = (wave << tokens_shift) + (uint32_t)(group >> p.slot_shift);
    r.head = group & ((1 << p.slot_shift) - 1);
    r.lane_in_group = lane & ((1 << p.group_shift) - 1);
    r.there = r.token < p.all_tokens;
    return r;
}

constexpr int kHeadsBlock = 256;

template <typename T, int V, int U, bool NORM>
__global__ __launch_bounds__(kHeadsBlock) void rotate_heads_kernel(HeadsArgs p)
{
    const Slot slot = slot_of(p, blockIdx.x * (kHeadsBlock / 64) + (threadIdx.x >> 6));
    if (!slot.there) return;  // whole groups leave: a group's lanes have one token
    Unit units[U];
#pragma unroll
    for (int k = 0; k < U; ++k) units[k] = unit_of<V>(p, slot.lane_in_group + (k << p.group_shift));
    const int64_t b = slot.token / p.tokens, t = slot.token % p.tokens;
    float c[U][V], s[U][V];
    make_turns<V, U>(p, units, b * p.position_stride[1] + t * p.position_stride[2], c, s);
    int head = slot.head + ((int)blockIdx.y << p.slot_shift);
    const int step = (int)gridDim.y << p.slot_shift;
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const T* x = static_cast<const T*>(p.x[which]) + b * p.x_stride[which][0] + t * p.x_stride[which][1];
        T* out = static_cast<T*>(p.out[which]) + (int64_t)slot.token * p.heads[which] * p.dim;
        Halves<T, V> w[U];
        if (NORM && head < p.heads[which]) {
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (units[k].there) w[k] = load_weight<T, V>(p, which, units[k]);
        }
        for (; head < p.heads[which]; head += step) {
            Halves<T, V> v[U];
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (!units[k].there) continue;
                v[k] = load_unit<T, V>(x + head * p.x_stride[which][2], units[k], p.interleaved);
                if (NORM) {
#pragma unroll
                    for (int e = 0; e < V; ++e) sum = __builtin_fmaf(v[k].a[e], v[k].a[e], __builtin_fmaf(v[k].b[e], v[k].b[e], sum));
                }
            }
            if (NORM) {
                const float r = 1.0f / sqrtf(__builtin_fmaf(group_sum(sum, p.group_shift), p.inv_dim, p.eps));
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
                if (units[k].pair >= 0) turn<T, V>(v[k], c[k], s[k]);
                store_unit<T, V>(out + (int64_t)head * p.dim, units[k], p.interleaved, v[k]);
            }
        }
        head -= p.heads[which];
    }
}

// With dy the gradient turned back, r = 1 / rms(x) and y = x r w:
//   dw = sum over tokens and heads of dy x r,   dx = r (w dy - x r^2 mean(x w dy)).
// The root is made again from x, which has to be read anyway.  A lane keeps its part of dw in registers over all heads and tokens
// that it takes; a workgroup leaves one row of sums, and sum_weight_grads_kernel adds the rows in their order: no atomics.
template <typename T, int V, int U>
__global__ __launch_bounds__(kHeadsBlock) void norm_rotate_heads_backward_kernel(HeadsArgs p, uint32_t waves)
{
    __shared__ float sums[2 * PS_MAX_HEAD_DIM];
    Halves<T, V> dw[2][U];
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) dw[which][k].a[e] = dw[which][k].b[e] = 0.0f;
    const int lane_in_group = threadIdx.x & ((1 << p.group_shift) - 1);
    Unit units[U];
#pragma unroll
    for (int k = 0; k < U; ++k) units[k] = unit_of<V>(p, lane_in_group + (k << p.group_shift));
    for (uint32_t wave = blockIdx.x * (kHeadsBlock / 64) + (threadIdx.x >> 6); wave < waves; wave += gridDim.x * (kHeadsBlock / 64)) {
        const Slot slot = slot_of(p, wave);
        if (!slot.there) continue;
        const int64_t b = slot.token / p.tokens, t = slot.token % p.tokens;
        float c[U][V], s[U][V];
        make_turns<V, U>(p, units, b * p.position_stride[1] + t * p.position_stride[2], c, s);
        int head = slot.head + ((int)blockIdx.y << p.slot_shift);
        const int step = (int)gridDim.y << p.slot_shift;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const T* x = static_cast<const T*>(p.x[which]) + b * p.x_stride[which][0] + t * p.x_stride[which][1];
            const T* g = static_cast<const T*>(p.grad[which]) + b * p.grad_stride[which][0] + t * p.grad_stride[which][1];
            T* out = static_cast<T*>(p.out[which]) + (int64_t)slot.token * p.heads[which] * p.dim;
            Halves<T, V> w[U];
            if (head < p.heads[which]) {
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (units[k].there) w[k] = load_weight<T, V>(p, which, units[k]);
            }
            for (; head < p.heads[which]; head += step) {
                Halves<T, V> v[U], d[U];
                float square = 0.0f, dot = 0.0f;
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    if (!units[k].there) continue;
                    v[k] = load_unit<T, V>(x + head * p.x_stride[which][2], units[k], p.interleaved);
                    d[k] = load_unit<T, V>(g + head * p.grad_stride[which][2], units[k], p.interleaved);
                    if (units[k].pair >= 0) turn<T, V>(d[k], c[k], s[k]);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        square = __builtin_fmaf(v[k].a[e], v[k].a[e], __builtin_fmaf(v[k].b[e], v[k].b[e], square));
                        dot = __builtin_fmaf(v[k].a[e] * w[k].a[e], d[k].a[e], __builtin_fmaf(v[k].b[e] * w[k].b[e], d[k].b[e], dot));
                    }
                }
                square = group_sum(square, p.group_shift);
                dot = group_sum(dot, p.group_shift);
                const float r = 1.0f / sqrtf(__builtin_fmaf(square, p.inv_dim, p.eps));
                const float back = r * r * (dot * p.inv_dim);
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    if (!units[k].there) continue;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float da = d[k].a[e], db = d[k].b[e];
                        dw[which][k].a[e] = __builtin_fmaf(da, v[k].a[e] * r, dw[which][k].a[e]);
                        dw[which][k].b[e] = __builtin_fmaf(db, v[k].b[e] * r, dw[which][k].b[e]);
                        d[k].a[e] = r * __builtin_fmaf(-v[k].a[e], back, w[k].a[e] * da);
                        d[k].b[e] = r * __builtin_fmaf(-v[k].b[e], back, w[k].b[e] * db);
                    }
                    store_unit<T, V>(out + (int64_t)head * p.dim, units[k], p.interleaved, d[k]);
                }
            }
            head -= p.heads[which];
        }
    }
    if (p.partial == nullptr) return;
    // groups of a wave, then the waves one after another
    for (int i = threadIdx.x; i < 2 * p.dim; i += kHeadsBlock) sums[i] = 0.0f;
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e)
                for (int m = 1 << p.group_shift; m < 64; m <<= 1) {
                    dw[which][k].a[e] += __shfl_xor(dw[which][k].a[e], m);
                    dw[which][k].b[e] += __shfl_xor(dw[which][k].b[e], m);
                }
    for (int wave = 0; wave < kHeadsBlock / 64; ++wave) {
        if ((int)(threadIdx.x >> 6) == wave && (threadIdx.x & 63) < (1u << p.group_shift)) {
#pragma unroll
            for (int which = 0; which < 2; ++which)
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    if (!units[k].there) continue;
                    const bool alternate = p.interleaved && units[k].pair >= 0;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        sums[which * p.dim + (alternate ? units[k].a + 2 * e : units[k].a + e)] += dw[which][k].a[e];
                        if (units[k].b >= 0) sums[which * p.dim + (alternate ? units[k].a + 2 * e + 1 : units[k].b + e)] += dw[which][k].b[e];
                    }
                }
        }
        __syncthreads();
    }
    float* row = p.partial + (int64_t)(blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.dim;
    for (int i = threadIdx.x; i < 2 * p.dim; i += kHeadsBlock) global(row)[i] = sums[i];
}

constexpr int kSumColumns = 32, kSumSlices = 32;

template <typename T>
__global__ __launch_bounds__(kSumColumns * kSumSlices) void sum_weight_grads_kernel(const float* partial, int rows, int dim, void* q_grad,
                                                                                   void* k_grad, bool f32)
{
    __shared__ float sums[kSumSlices][kSumColumns + 1];
    const int column = blockIdx.x * kSumColumns + (threadIdx.x % kSumColumns), slice = threadIdx.x / kSumColumns;
    float sum = 0.0f;
    if (column < 2 * dim)
        for (int r = slice; r < rows; r += kSumSlices) sum += global(partial)[(int64_t)r * 2 * dim + column];
    sums[slice][threadIdx.x % kSumColumns] = sum;
    __syncthreads();
    if (slice != 0 || column >= 2 * dim) return;
    sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kSumSlices; ++k) sum += sums[k][threadIdx.x];
    void* out = column < dim ? q_grad : k_grad;
    const int at = column < dim ? column : column - dim;
    if (out == nullptr) return;
    if (f32)
        global(static_cast<float*>(out))[at] = sum;
    else
        global(static_cast<T*>(out))[at] = from_float<T>(sum);
}

}  // namespace

#endif  // PS_ROTARY_H
