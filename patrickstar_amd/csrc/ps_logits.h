// Kernels of ps_top_logits, ps_distill_loss and ps_distill_loss_backward.
//
// One workgroup takes a row of logits at a time.  A row that fits is loaded once, all of its loads in flight together, and stays in
// the workgroup's registers (in its own type, NV 16-byte vectors a thread) while maximum, sums and gradient are made from it;
// a longer one (NV = 0) is read again for each of them.
#ifndef PS_LOGITS_H
#define PS_LOGITS_H

#include "ps_vec.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// ---------------------------------------------------------------------------------------------------- a row and its parts

// The elements of a row: up to VE - 1 in front of the first 16-byte boundary, whole vectors, up to VE - 1 behind the last one.  The
// ones at the ends are a thread's own each ("lone").
template <typename T>
struct RowShape {
    static constexpr int VE = 16 / (int)sizeof(T);
    const T* row;
    int head, vectors, vocab;

    __device__ __forceinline__ RowShape(const T* r, int v) : row(r), vocab(v)
    {
        head = (int)((16 - (reinterpret_cast<uintptr_t>(r) & 15)) & 15) / (int)sizeof(T);
        head = head < v ? head : v;
        vectors = (v - head) / VE;
    }
    __device__ __forceinline__ int element_of(int vector) const { return head + vector * VE; }
    // place of a thread's lone element, or -1
    __device__ __forceinline__ int lone_of(int thread) const
    {
        if (thread < head) return thread;
        const int at = thread + vectors * VE;
        return at < vocab ? at : -1;
    }
};

template <typename T>
struct RowVec {
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
    // for rows of the gradient, which may start at any element
    typedef type __attribute__((aligned(sizeof(T)))) loose;
};

template <typename T>
__device__ __forceinline__ void store_loose(T* p, typename RowVec<T>::type v)
{
    *(__attribute__((address_space(1))) typename RowVec<T>::loose*)(p) = v;
}

template <typename T>
__device__ __forceinline__ T lowest();
template <>
__device__ __forceinline__ half_t lowest<half_t>()
{
    return (half_t)-__builtin_inff();
}
template <>
__device__ __forceinline__ bf16_t lowest<bf16_t>()
{
    return (bf16_t)-__builtin_inff();
}
template <>
__device__ __forceinline__ float lowest<float>()
{
    return -__builtin_inff();
}

// Calls f(values, first element, count) for the thread's vectors and its lone element; `keep` holds them between calls if NV > 0.
template <typename T, int NV, int BLOCK>
struct RowData {
    typedef typename RowVec<T>::type vec;
    static constexpr int VE = RowShape<T>::VE;
    vec kept[NV > 0 ? NV : 1];
    T lone;
    int lone_at;

    __device__ __forceinline__ void load(const RowShape<T>& s)
    {
        lone_at = s.lone_of(threadIdx.x);
        if (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int v = i * BLOCK + (int)threadIdx.x;
                if (v < s.vectors) {
                    kept[i] = *global(reinterpret_cast<const vec*>(s.row + s.element_of(v)));
                } else {
#pragma unroll
                    for (int e = 0; e < VE; ++e) kept[i][e] = lowest<T>();
                }
            }
        }
        lone = lone_at >= 0 ? *global(s.row + lone_at) : lowest<T>();
    }
    // f(vec, first element) for every vector of the thread that is there, then g(value, element)
    template <typename F, typename G>
    __device__ __forceinline__ void each(const RowShape<T>& s, F f, G g) const
    {
        if (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int v = i * BLOCK + (int)threadIdx.x;
                if (v < s.vectors) f(kept[i], s.element_of(v));
            }
        } else {
            for (int v = threadIdx.x; v < s.vectors; v += BLOCK) {
                const vec x = *global(reinterpret_cast<const vec*>(s.row + s.element_of(v)));
                f(x, s.element_of(v));
            }
        }
        if (lone_at >= 0) g(lone, lone_at);
    }
};

// ------------------------------------------------------------------------------------------------------------ reductions

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) {
        const uint32_t o = __shfl_xor(v, m);
        v = o > v ? o : v;
    }
    return v;
}
__device__ __forceinline__ int wave_sum(int v)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// Every thread gets the result.  Each use needs LDS of its own, or a barrier between the uses.
template <int BLOCK, typename N>
__device__ __forceinline__ N block_max(N v, N* lds)
{
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    N r = lds[0];
#pragma unroll
    for (int k = 1; k < BLOCK / 64; ++k) r = lds[k] > r ? lds[k] : r;
    return r;
}
template <int BLOCK, typename N>
__device__ __forceinline__ N block_sum(N v, N* lds)
{
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    N r = lds[0];
#pragma unroll
    for (int k = 1; k < BLOCK / 64; ++k) r += lds[k];
    return r;
}

// ------------------------------------------------------------------------------------------------------------ top logits

struct TopArgs {
    const void* logits;
    void* values;
    int32_t* ids;
    float* lse;
    int64_t rows, row_stride;
    int vocab, k;
    float factor, temperature;  // log2(e) / temperature
};

// Whole numbers in the order of the values: zeros of both signs alike, NaN above everything, never 0.
__device__ __forceinline__ uint32_t order_of(float x)
{
    if (x != x) return 0xFFFFFFFFu;
    uint32_t b;
    x = x + 0.0f;  // -0 -> +0
    __builtin_memcpy(&b, &x, 4);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float number_of(uint32_t order)
{
    const uint32_t b = order & 0x80000000u ? order & 0x7FFFFFFFu : ~order;
    float x;
    __builtin_memcpy(&x, &b, 4);
    return x;  // (NaN: 0x7FFFFFFF)
}

constexpr int kTopCandidates = 2048;

// 1. A thread's largest element; the k-th largest of these bounds the k-th largest of the row from below (k threads have one at
//    least as large), and few elements reach it.  2. Those that do go to LDS; there, an element's place is the number of larger ones.
// Where too many reach the bound (long runs of equal logits), the k-th largest (order, place) is found bit by bit: all are
// different, so exactly k reach it.
template <typename T, int NV, int BLOCK>
__global__ __launch_bounds__(BLOCK) void top_logits_kernel(TopArgs p)
{
    typedef typename RowVec<T>::type vec;
    constexpr int VE = RowShape<T>::VE;
    __shared__ uint64_t found[kTopCandidates];
    __shared__ uint32_t largest[BLOCK];
    __shared__ uint32_t lds_max[BLOCK / 64];
    __shared__ float lds_sum[BLOCK / 64];
    __shared__ int lds_count[2][BLOCK / 64];
    __shared__ uint32_t bound_at;
    __shared__ int n_found;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* row = static_cast<const T*>(p.logits) + r * p.row_stride;
        const RowShape<T> shape(row, p.vocab);
        RowData<T, NV, BLOCK> data;
        data.load(shape);
        uint32_t mine = 0;
        data.each(
            shape,
            [&](const vec& v, int) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const uint32_t o = order_of(to_float<T>(v[e]));
                    mine = o > mine ? o : mine;
                }
            },
            [&](T x, int) {
                const uint32_t o = order_of(to_float<T>(x));
                mine = o > mine ? o : mine;
            });
        largest[threadIdx.x] = mine;
        if (threadIdx.x == 0) n_found = 0;
        const float m = number_of(block_max<BLOCK>(mine, lds_max));  // (a barrier: `largest` is there)
        // the sum of exponentials; NaN wherever a logit is NaN or +inf
        float sum = 0.0f;
        data.each(
            shape,
            [&](const vec& v, int) {
#pragma unroll
                for (int e = 0; e < VE; ++e) sum += exp2_fast((to_float<T>(v[e]) - m) * p.factor);
            },
            [&](T x, int) { sum += exp2_fast((to_float<T>(x) - m) * p.factor); });
        if (threadIdx.x < 64) {
            // the k-th largest of the threads' largest: the greatest bound that k of them reach, bit by bit
            uint32_t bound = 0;
            if (p.k <= BLOCK) {
                uint32_t all[BLOCK / 64];
#pragma unroll
                for (int i = 0; i < BLOCK / 64; ++i) all[i] = largest[i * 64 + threadIdx.x];
                // bits below the type's own are alike in all numbers of a sign; of fp32 the last ten are left at 0 (a lower bound)
                constexpr int kLowBit = sizeof(T) == 4 ? 10 : __is_same(T, half_t) ? 13 : 16;
                for (int bit = 31; bit >= kLowBit; --bit) {
                    const uint32_t next = bound | 1u << bit;
                    int n = 0;
#pragma unroll
                    for (int i = 0; i < BLOCK / 64; ++i) n += __popcll(__ballot(all[i] >= next));
                    if (n >= p.k) bound = next;
                }
            }
            if (threadIdx.x == 0) bound_at = bound;
        }
        sum = block_sum<BLOCK>(sum, lds_sum);  // (a barrier: the bound is there)
        const uint32_t bound = bound_at;
        if (threadIdx.x == 0) {
            const bool finite = m - m == 0.0f;  // a row of -inf alone has no mass, one with +inf all of it there; NaN stays
            const float lse = finite ? m / p.temperature + __builtin_amdgcn_logf(sum) * kLn2 : m;
            *global(p.lse + r) = lse;
        }
        auto keep = [&](uint64_t entry) {
            const int at = atomicAdd(&n_found, 1);
            if (at < kTopCandidates) found[at] = entry;
        };
        auto entry_of = [](float x, int at) { return (uint64_t)order_of(x) << 32 | (0xFFFFFFFFu - (uint32_t)at); };
        if (mine >= bound && mine != 0) {
            data.each(
                shape,
                [&](const vec& v, int at) {
#pragma unroll
                    for (int e = 0; e < VE; ++e)
                        if (order_of(to_float<T>(v[e])) >= bound) keep(entry_of(to_float<T>(v[e]), at + e));
                },
                [&](T x, int at) {
                    if (order_of(to_float<T>(x)) >= bound) keep(entry_of(to_float<T>(x), at));
                });
        }
        __syncthreads();
        int n = n_found;
        if (n > kTopCandidates) {
            uint64_t least = 0;
            int turn = 0;
            for (int bit = 63; bit >= 0; --bit) {
                const uint64_t next = least | 1ull << bit;
                int count = 0;
                data.each(
                    shape,
                    [&](const vec& v, int at) {
#pragma unroll
                        for (int e = 0; e < VE; ++e) count += entry_of(to_float<T>(v[e]), at + e) >= next;
                    },
                    [&](T x, int at) { count += entry_of(to_float<T>(x), at) >= next; });
                count = block_sum<BLOCK>(count, lds_count[turn]);
                turn ^= 1;
                if (count >= p.k) least = next;
                if (count == p.k) break;
            }
            if (threadIdx.x == 0) n_found = 0;
            __syncthreads();
            data.each(
                shape,
                [&](const vec& v, int at) {
#pragma unroll
                    for (int e = 0; e < VE; ++e)
                        if (entry_of(to_float<T>(v[e]), at + e) >= least) keep(entry_of(to_float<T>(v[e]), at + e));
                },
                [&](T x, int at) {
                    if (entry_of(to_float<T>(x), at) >= least) keep(entry_of(to_float<T>(x), at));
                });
            __syncthreads();
            n = n_found;
        }
        for (int i = threadIdx.x; i < n; i += BLOCK) {
            const uint64_t mine_entry = found[i];
            int place = 0;
            for (int j = 0; j < n; ++j) place += found[j] > mine_entry;
            if (place < p.k) {
                const uint32_t at = 0xFFFFFFFFu - (uint32_t)mine_entry;
                *global(p.ids + r * p.k + place) = (int32_t)at;
                *global(static_cast<T*>(p.values) + r * p.k + place) = *global(row + at);
            }
        }
        __syncthreads();  // before the next row's candidates
    }
}

// ------------------------------------------------------------------------------------------------------------ distillation

struct DistillArgs {
    const void* logits;
    const void* ids;
    const void* values;
    const float* teacher_lse;
    const void* labels;
    float* row_loss;
    float* stats;
    const float* denominator;
    void* grad;
    const float* upstream;
    float* upstream_used;
    int64_t rows, row_stride, ids_stride, values_stride, upstream_stride;
    int64_t ignore_index;
    int vocab, k;
    int values_dtype;
    float temperature, label_weight, upstream_value;
    bool ids_64, labels_64;
};

__device__ __forceinline__ int64_t whole_at(const void* p, int64_t at, bool is64)
{
    return is64 ? *global(static_cast<const int64_t*>(p) + at) : (int64_t)*global(static_cast<const int32_t*>(p) + at);
}
__device__ __forceinline__ float value_at(const void* p, int64_t at, int dtype)
{
    if (dtype == PS_F32) return *global(static_cast<const float*>(p) + at);
    if (dtype == PS_BF16) return (float)*global(static_cast<const bf16_t*>(p) + at);
    return (float)*global(static_cast<const half_t*>(p) + at);
}

// What a row's gradient is made from.
struct RowStats {
    float m;       // largest logit
    float inv_s;   // 1 / sum of exp((z - m) / temperature)
    float coef;    // a softmax's share in the gradient off the list: 1 - rest / q_rest, or the list's mass
    float inv_s1;  // 1 / sum of exp(z - m)
};

// The teacher's list in LDS: ids, probabilities.  Returns through `mass` their sum (every thread).
template <int BLOCK>
__device__ __forceinline__ void load_list(const DistillArgs& p, int64_t r, int* ids, float* prob, float* lds_a, float* lds_b, float& mass)
{
    float top = -__builtin_inff();
    for (int i = threadIdx.x; i < p.k; i += BLOCK) {
        const int64_t id = whole_at(p.ids, r * p.ids_stride + i, p.ids_64);
        const float v = value_at(p.values, r * p.values_stride + i, p.values_dtype) / p.temperature;
        ids[i] = id < 0 ? -1 : id < p.vocab ? (int)id : -2;  // -2: beyond the vocabulary
        prob[i] = v;
        if (id >= 0) top = fmaxf(top, v);
    }
    const bool rest = p.teacher_lse != nullptr;
    if (rest)
        top = *global(p.teacher_lse + r);
    else
        top = block_max<BLOCK, float>(top, lds_a);
    float sum = 0.0f;
    for (int i = threadIdx.x; i < p.k; i += BLOCK) {  // (a thread's own entries)
        const float e = ids[i] == -1 ? 0.0f : expf(prob[i] - top);
        prob[i] = e;
        sum += e;
    }
    mass = block_sum<BLOCK>(sum, lds_b);
    if (!rest) {
        const float scale = mass > 0.0f ? 1.0f / mass : mass == mass ? 0.0f : mass;
        for (int i = threadIdx.x; i < p.k; i += BLOCK) prob[i] *= scale;
        mass = mass > 0.0f ? 1.0f : mass;
    }
    __syncthreads();
}

// The row's gradient, from registers or memory: list entries and label after everything else, over it.
template <typename T, int NV, int BLOCK>
__device__ __forceinline__ void write_gradient(const DistillArgs& p, int64_t r, const RowShape<T>& shape, const RowData<T, NV, BLOCK>& data,
                                               const RowStats& s, float factor, const int* ids, const float* prob, int64_t label)
{
    typedef typename RowVec<T>::type vec;
    constexpr int VE = RowShape<T>::VE;
    T* out = static_cast<T*>(p.grad) + r * (int64_t)p.vocab;
    const float c = kLog2e / p.temperature;
    const float soft = factor * (1.0f - p.label_weight) * p.temperature * s.inv_s;
    const float hard = factor * p.label_weight * s.inv_s1;
    const float off = soft * s.coef;
    const bool soft_there = p.label_weight != 1.0f, hard_there = p.label_weight != 0.0f;
    const bool both = soft_there && hard_there;
    const float c1 = soft_there ? c : kLog2e, a1 = soft_there ? off : hard;
    if (both) {
        data.each(
            shape,
            [&](const vec& v, int at) {
                vec g;
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float d = to_float<T>(v[e]) - s.m;
                    g[e] = from_float<T>(__builtin_fmaf(exp2_fast(d * c), off, exp2_fast(d * kLog2e) * hard));
                }
                store_loose<T>(out + at, g);
            },
            [&](T x, int at) {
                const float d = to_float<T>(x) - s.m;
                *global(out + at) = from_float<T>(__builtin_fmaf(exp2_fast(d * c), off, exp2_fast(d * kLog2e) * hard));
            });
    } else {
        data.each(
            shape,
            [&](const vec& v, int at) {
                vec g;
#pragma unroll
                for (int e = 0; e < VE; ++e) g[e] = from_float<T>(exp2_fast((to_float<T>(v[e]) - s.m) * c1) * a1);
                store_loose<T>(out + at, g);
            },
            [&](T x, int at) { *global(out + at) = from_float<T>(exp2_fast((to_float<T>(x) - s.m) * c1) * a1); });
    }
    __syncthreads();
    const float mass_factor = p.teacher_lse != nullptr ? 1.0f : s.coef;
    const float given = factor * (1.0f - p.label_weight) * p.temperature;
    if (soft_there) {
        for (int i = threadIdx.x; i < p.k; i += BLOCK) {
            const int id = ids[i];
            if (id < 0) continue;
            const float d = to_float<T>(*global(shape.row + id)) - s.m;
            float g = exp2_fast(d * c) * soft * mass_factor - given * prob[i];
            if (hard_there) g += exp2_fast(d * kLog2e) * hard - (id == label ? factor * p.label_weight : 0.0f);
            *global(out + id) = from_float<T>(g);
        }
    }
    if (hard_there) {
        // the label, unless it is on the list: the thread of its entry has written it
        bool listed = false;
        if (soft_there)
            for (int i = threadIdx.x; i < p.k; i += BLOCK) listed |= ids[i] == label;
        if (!__syncthreads_or(listed) && threadIdx.x == 0 && label >= 0 && label < p.vocab) {
            const float d = to_float<T>(*global(shape.row + label)) - s.m;
            float g = exp2_fast(d * kLog2e) * hard - factor * p.label_weight;
            if (soft_there) g += exp2_fast(d * c) * off;
            *global(out + label) = from_float<T>(g);
        }
    }
}

template <typename T, int NV, int BLOCK>
__device__ __forceinline__ void write_zeros(const DistillArgs& p, int64_t r, const RowShape<T>& shape)
{
    typedef typename RowVec<T>::type vec;
    T* out = static_cast<T*>(p.grad) + r * (int64_t)p.vocab;
    vec zero;
#pragma unroll
    for (int e = 0; e < RowShape<T>::VE; ++e) zero[e] = (T)0.0f;
    for (int v = threadIdx.x; v < shape.vectors; v += BLOCK) store_loose<T>(out + shape.element_of(v), zero);
    const int lone = shape.lone_of(threadIdx.x);
    if (lone >= 0) *global(out + lone) = (T)0.0f;
}

// Dynamic LDS: a bit for every token of the vocabulary (is it on the list?), then the list's ids and probabilities.
template <typename T, int NV, int BLOCK>
__global__ __launch_bounds__(BLOCK) void distill_loss_kernel(DistillArgs p)
{
    typedef typename RowVec<T>::type vec;
    constexpr int VE = RowShape<T>::VE;
    extern __shared__ uint32_t dynamic[];
    __shared__ float lds[6][BLOCK / 64];
    const int words = (p.vocab + 31) / 32;
    uint32_t* member = dynamic;
    int* ids = reinterpret_cast<int*>(dynamic + words);
    float* prob = reinterpret_cast<float*>(dynamic + words + p.k);
    const bool rest = p.teacher_lse != nullptr;
    const bool soft = p.label_weight != 1.0f, hard = p.label_weight != 0.0f;
    const float c = kLog2e / p.temperature;
    const float upstream = p.upstream ? *global(p.upstream) : p.upstream_value;
    if (p.upstream_used && blockIdx.x == 0 && threadIdx.x == 0) *global(p.upstream_used) = upstream;
    const float inv_count = p.denominator ? 1.0f / *global(p.denominator) : 1.0f;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const RowShape<T> shape(static_cast<const T*>(p.logits) + r * p.row_stride, p.vocab);
        int64_t label = -1;
        bool wrong = false;
        if (p.labels) {
            label = whole_at(p.labels, r, p.labels_64);
            if (label == p.ignore_index) {
                if (threadIdx.x == 0) {
                    *global(p.row_loss + r) = 0.0f;
                    if (p.stats)
                        for (int i = 0; i < 4; ++i) *global(p.stats + 4 * r + i) = 0.0f;
                }
                if (p.grad) write_zeros<T, NV, BLOCK>(p, r, shape);
                continue;
            }
            if (hard) wrong = label < 0 || label >= p.vocab;
        }
        RowData<T, NV, BLOCK> data;
        data.load(shape);
        for (int i = threadIdx.x; i < words; i += BLOCK) member[i] = 0;
        float mass;
        load_list<BLOCK>(p, r, ids, prob, lds[0], lds[1], mass);
        for (int i = threadIdx.x; i < p.k; i += BLOCK) {
            const int id = ids[i];
            if (id >= 0)
                wrong |= (atomicOr(&member[id >> 5], 1u << (id & 31)) >> (id & 31)) & 1;
            else
                wrong |= id == -2;
        }
        float m = -__builtin_inff();
        data.each(
            shape,
            [&](const vec& v, int) {
#pragma unroll
                for (int e = 0; e < VE; ++e) m = fmaxf(m, to_float<T>(v[e]));
            },
            [&](T x, int) { m = fmaxf(m, to_float<T>(x)); });
        m = block_max<BLOCK, float>(m, lds[2]);  // (a barrier: the members are there)
        float sum = 0.0f, sum_rest = 0.0f, sum1 = 0.0f;
        const float first = soft ? c : kLog2e;
        data.each(
            shape,
            [&](const vec& v, int at) {
                float part = 0.0f;
                float x[VE];
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    x[e] = exp2_fast((to_float<T>(v[e]) - m) * first);
                    part += x[e];
                }
                sum += part;
                if (rest) {
                    // the vector's members: VE bits that may lie in two words
                    const uint32_t lo = member[at >> 5], hi = member[(at + VE - 1) >> 5];
                    const uint32_t bits = (uint32_t)(((uint64_t)hi << 32 | lo) >> (at & 31)) & ((1u << VE) - 1);
                    if (bits) {
                        part = 0.0f;
#pragma unroll
                        for (int e = 0; e < VE; ++e) part += bits >> e & 1 ? 0.0f : x[e];
                    }
                    sum_rest += part;
                }
                if (soft && hard) {
#pragma unroll
                    for (int e = 0; e < VE; ++e) sum1 += exp2_fast((to_float<T>(v[e]) - m) * kLog2e);
                }
            },
            [&](T x, int at) {
                const float e = exp2_fast((to_float<T>(x) - m) * first);
                sum += e;
                if (rest && !(member[at >> 5] >> (at & 31) & 1)) sum_rest += e;
                if (soft && hard) sum1 += exp2_fast((to_float<T>(x) - m) * kLog2e);
            });
        // the list's part of the divergence does not need the sums: sum p (log p - z) and sum p
        float term = 0.0f;
        if (soft) {
            for (int i = threadIdx.x; i < p.k; i += BLOCK) {
                const float pr = prob[i];
                if (ids[i] >= 0 && pr != 0.0f)
                    term = __builtin_fmaf(pr, logf(pr) - (to_float<T>(*global(shape.row + ids[i])) - m) / p.temperature, term);
            }
        }
        sum = wave_sum(sum), sum_rest = wave_sum(sum_rest), sum1 = wave_sum(sum1), term = wave_sum(term);
        if ((threadIdx.x & 63) == 0) {
            lds[0][threadIdx.x >> 6] = sum;
            lds[1][threadIdx.x >> 6] = sum_rest;
            lds[3][threadIdx.x >> 6] = sum1;
            lds[4][threadIdx.x >> 6] = term;
        }
        wrong = __syncthreads_or(wrong);
        sum = sum_rest = sum1 = term = 0.0f;
#pragma unroll
        for (int w = 0; w < BLOCK / 64; ++w) {
            sum += lds[0][w];
            sum_rest += lds[1][w];
            sum1 += lds[3][w];
            term += lds[4][w];
        }
        if (!soft) sum1 = sum;
        if (wrong) sum = sum1 = __builtin_nanf("");
        RowStats s;
        s.m = m;
        s.inv_s = soft ? 1.0f / sum : 0.0f;
        s.inv_s1 = hard ? 1.0f / sum1 : 0.0f;
        const float p_rest = fmaxf(1.0f - mass, 0.0f), q_rest = sum_rest * s.inv_s;
        s.coef = rest ? (p_rest == 0.0f ? 1.0f : 1.0f - p_rest / q_rest) : mass;
        if (threadIdx.x == 0) {
            float loss = 0.0f;
            if (soft) {
                float kl = __builtin_fmaf(mass, logf(sum), term);  // + sum p log s
                if (rest && p_rest > 0.0f) kl = __builtin_fmaf(p_rest, logf(p_rest) - logf(q_rest), kl);
                loss = (1.0f - p.label_weight) * p.temperature * p.temperature * kl;
            }
            if (hard) {
                const float z = wrong ? m : to_float<T>(*global(shape.row + label));
                loss = __builtin_fmaf(p.label_weight, logf(sum1) - (z - m), loss);
            }
            *global(p.row_loss + r) = loss;
            if (p.stats) {
                *global(p.stats + 4 * r) = s.m;
                *global(p.stats + 4 * r + 1) = s.inv_s;
                *global(p.stats + 4 * r + 2) = s.coef;
                *global(p.stats + 4 * r + 3) = s.inv_s1;
            }
        }
        if (p.grad) write_gradient<T, NV, BLOCK>(p, r, shape, data, s, upstream * inv_count, ids, prob, label);
        __syncthreads();  // before the next row's list
    }
}

template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void distill_backward_kernel(DistillArgs p)
{
    extern __shared__ uint32_t dynamic[];
    __shared__ float lds[2][BLOCK / 64];
    // the gradient that the forward pass made is at this very factor
    if (p.upstream_used && *global(p.upstream) == *global(p.upstream_used)) return;
    int* ids = reinterpret_cast<int*>(dynamic);
    float* prob = reinterpret_cast<float*>(dynamic + p.k);
    const float inv_count = p.denominator ? 1.0f / *global(p.denominator) : 1.0f;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const RowShape<T> shape(static_cast<const T*>(p.logits) + r * p.row_stride, p.vocab);
        const int64_t label = p.labels ? whole_at(p.labels, r, p.labels_64) : -1;
        if (p.labels && label == p.ignore_index) {
            write_zeros<T, 0, BLOCK>(p, r, shape);
            continue;
        }
        RowStats s;
        s.m = *global(p.stats + 4 * r);
        s.inv_s = *global(p.stats + 4 * r + 1);
        s.coef = *global(p.stats + 4 * r + 2);
        s.inv_s1 = *global(p.stats + 4 * r + 3);
        float mass;
        load_list<BLOCK>(p, r, ids, prob, lds[0], lds[1], mass);
        RowData<T, 0, BLOCK> data;
        data.load(shape);
        write_gradient<T, 0, BLOCK>(p, r, shape, data, s, *global(p.upstream + r * p.upstream_stride) * inv_count, ids, prob, label);
        __syncthreads();
    }
}

// One workgroup: how many rows count (at least 1).
__global__ __launch_bounds__(1024) void count_rows_kernel(const void* labels, bool is64, int64_t rows, int64_t ignore_index, float* out)
{
    __shared__ int lds[16];
    int n = 0;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) n += labels == nullptr || whole_at(labels, r, is64) != ignore_index;
    n = block_sum<1024>(n, lds);
    if (threadIdx.x == 0) *global(out) = (float)(n > 0 ? n : 1);
}

// One workgroup, a fixed order: the same rows give the same loss.  In 64 bits: a row more costs nothing here.
__global__ __launch_bounds__(1024) void sum_rows_kernel(const float* row_loss, int64_t rows, const float* denominator, float* out)
{
    __shared__ double lds[1024];
    double sum = 0.0;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) sum += (double)*global(row_loss + r);
    lds[threadIdx.x] = sum;
    for (int n = 512; n; n >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < n) lds[threadIdx.x] += lds[threadIdx.x + n];
    }
    if (threadIdx.x == 0) *global(out) = (float)(lds[0] / (denominator ? (double)*global(denominator) : 1.0));
}

}  // namespace

#endif  // PS_LOGITS_H
