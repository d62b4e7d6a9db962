// Kernels of ps_top_logits, ps_distill_loss and ps_distill_loss_backward.
//
// One workgroup takes a row of logits at a time.  A row that fits is loaded once, all of its loads in flight together, and stays in
// the workgroup's registers (in its own type, NV 16-byte vectors a thread) while maximum, sums and gradient are made from it;
// a longer one (NV = 0) is read again for each of them (by ps_top_logits once).
//
// Memory bounds it as long as little is done for a logit: at 16 bits each, a CU has 13 operations for one while it is read.  So a
// softmax takes a fused multiply-add, the exponential and an addition; the maximum half an operation; whatever is needed once a row or
// for a list is kept away from the loops over the row.  Rows of an odd vocabulary start at any element: vectors begin at the first
// 16-byte boundary (16-byte reads from odd elements reach 4.8 TB/s, from boundaries 6.1).  Registers decide how many rows a CU works
// on at a time, and that hides what a row waits for: values derived from the row are hidden from the compiler, which would keep them
// (distillation of 8192 x 50257 took 585 us with, 341 without), and loops over rows too (their invariants took 20 to 40 registers).
// Measured (GPU time):
//   top 64 of 8192 x 50257 fp16                                  155 us, 0.83 GB, 5.3 TB/s (133 us for reading it)
//   top 200 of 500 x 200000 fp32                                  87 us, 0.40 GB, 4.6 TB/s
//   distillation of 8192 x 50257 fp16, a tenth ignored, loss and gradient  330 us, 1.56 GB, 4.7 TB/s (a copy of such rows: 4.8)
//   the loss alone of 4096 x 30522 bf16, a fifth ignored          50 us, 0.20 GB, 4.0 TB/s
#ifndef PS_LOGITS_H
#define PS_LOGITS_H

#include "ps_vec.h"

namespace {

// (of lambdas that the kernels call in several places: left to itself the compiler keeps their captures in memory)
#define PS_INLINE __attribute__((always_inline))

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Softmaxes are taken as exp2(z c - m c), c = log2(e) / temperature and m the row's largest logit: one fused multiply-add in front of
// the exponential, whose rounding of m c is the same for the whole row and falls out of every quotient.  Where m c would overflow
// (a row of the type's lowest value, say), two logits that differ at all differ by 2^-24 m at least, so that the smaller one has no
// mass, and a smaller factor gives the same softmax.
__device__ __forceinline__ float row_factor(float m, float c)
{
    const float size = fabsf(m);
    return size * c < 1e37f || size == __builtin_inff() ? c : 1e36f / size;
}

// log(sum(exp(z / temperature))) from the row's sum of exponentials under m, which are exp2(bias) times too large.  Rows are compared by
// differences of these, which are far smaller than they are: once a row, in 64 bits.
__device__ __forceinline__ double log_sum(float m, float bias, double sum, double temperature)
{
    return (double)m / temperature + (log(sum) - 0.6931471805599453 * (double)bias);
}

// ---------------------------------------------------------------------------------------------------- a row and its parts

typedef uint32_t raw_t __attribute__((ext_vector_type(4)));  // a vector of a row as it lies in memory

template <typename T>
struct RowVec {
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
    // for rows of the gradient, which may start at any element
    typedef type __attribute__((aligned(sizeof(T)))) loose;
};

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
    // (a 32-bit offset from an address that is the same for the whole wave: no 64-bit address in registers)
    __device__ __forceinline__ raw_t vector_at(int vector) const
    {
        return *global(reinterpret_cast<const raw_t*>(reinterpret_cast<const char*>(row + head) + (uint32_t)vector * 16u));
    }
    // the same vector of another row with this shape, which may start at any element
    __device__ __forceinline__ void store(T* other, int vector, typename RowVec<T>::type v) const
    {
        char* at = reinterpret_cast<char*>(other + head) + (uint32_t)vector * 16u;
        *(__attribute__((address_space(1))) typename RowVec<T>::loose*)(at) = v;
    }
    // place of a thread's lone element, or -1
    __device__ __forceinline__ int lone_of(int thread) const
    {
        if (thread < head) return thread;
        const int at = thread + vectors * VE;
        return at < vocab ? at : -1;
    }
};

// The thread's number, such that what is computed from it is not kept in registers from one use of the row to the next.
__device__ __forceinline__ int fresh_thread()
{
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// The largest of the elements given.  NaN is passed over: the sums behind it find it.  (Written as instructions: the compiler puts
// a canonicalization of every operand in front of its own maximum, which triples the work.)
template <typename T>
struct Largest {
    float top = -__builtin_inff();

    __device__ __forceinline__ void add(raw_t v)
    {
        if constexpr (sizeof(T) == 4) {
            asm("v_max3_f32 %0, %0, %1, %2" : "+v"(top) : "v"(v[0]), "v"(v[1]));
            asm("v_max3_f32 %0, %0, %1, %2" : "+v"(top) : "v"(v[2]), "v"(v[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) asm("v_max3_f32 %0, %0, %1, %2" : "+v"(top) : "v"(v[i] << 16), "v"(v[i] & 0xFFFF0000u));
        }
    }
    __device__ __forceinline__ void add(T x) { top = fmaxf(top, to_float<T>(x)); }
    __device__ __forceinline__ float get() const { return top; }
};
template <>
struct Largest<half_t> {
    uint32_t two = 0xFC00FC00u;  // -inf, -inf
    float top = -__builtin_inff();

    __device__ __forceinline__ void add(raw_t v)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("v_pk_max_f16 %0, %0, %1" : "+v"(two) : "v"(v[i]));
    }
    __device__ __forceinline__ void add(half_t x) { top = fmaxf(top, (float)x); }
    __device__ __forceinline__ float get() const
    {
        typedef half_t half2 __attribute__((ext_vector_type(2)));
        const half2 h = __builtin_bit_cast(half2, two);
        return fmaxf(top, fmaxf((float)h[0], (float)h[1]));
    }
};

// A thread's part of a row: its vectors (in registers if NV > 0) and its lone element.
template <typename T, int NV, int BLOCK>
struct RowData {
    typedef typename RowVec<T>::type vec;
    static constexpr int VE = RowShape<T>::VE;
    raw_t kept[NV > 0 ? NV : 1];
    T lone;
    int lone_at;

    __device__ __forceinline__ void load(const RowShape<T>& s)
    {
        lone_at = s.lone_of(threadIdx.x);
        lone = (T)0.0f;
        if (lone_at >= 0) lone = *global(s.row + lone_at);
        const int thread = fresh_thread();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int v = i * BLOCK + thread;
            if (v < s.vectors) kept[i] = s.vector_at(v);
        }
    }
    // What is made of the vectors in one use (their elements in 32 bits) shall not be kept in registers for the next one.
    __device__ __forceinline__ void hide()
    {
#pragma unroll
        for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(kept[i]));
    }
    // f(raw vector, its number) for every vector of the thread, then g(value, element) for its lone one
    template <typename F, typename G>
    __device__ __forceinline__ void each_raw(const RowShape<T>& s, F f, G g) const
    {
        if (NV > 0) {
            const int thread = fresh_thread();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int v = i * BLOCK + thread;
                if (v < s.vectors) f(kept[i], v);
                __builtin_amdgcn_sched_barrier(0);  // vectors worked on side by side would take more registers than there are
            }
        } else {
            for (int v = threadIdx.x; v < s.vectors; v += BLOCK) {
                f(s.vector_at(v), v);
            }
        }
        if (lone_at >= 0) g(lone, lone_at);
    }
    template <typename F, typename G>
    __device__ __forceinline__ void each(const RowShape<T>& s, F f, G g) const
    {
        each_raw(s, [&](raw_t x, int v) PS_INLINE { f(__builtin_bit_cast(vec, x), v); }, g);
    }
    __device__ __forceinline__ float largest(const RowShape<T>& s) const
    {
        Largest<T> top;
        each_raw(s, [&](raw_t x, int) PS_INLINE { top.add(x); }, [&](T x, int) PS_INLINE { top.add(x); });
        return top.get();
    }
};

// ------------------------------------------------------------------------------------------------------------ reductions

// Of all lanes of a wave, the same in every one: within 16 lanes by moves between lanes as part of the operation, then of the four
// sixteens.
template <typename N, typename F>
__device__ __forceinline__ N wave_fold(N v, F f)
{
    v = f(v, moved<0xB1>(v));   // the other of a pair
    v = f(v, moved<0x4E>(v));   // the other pair of four
    v = f(v, moved<0x141>(v));  // mirrored in eight: fours are alike by now
    v = f(v, moved<0x140>(v));  // mirrored in sixteen
    return f(f(of_lane(v, 0), of_lane(v, 16)), f(of_lane(v, 32), of_lane(v, 48)));
}
template <typename N>
__device__ __forceinline__ N wave_sum(N v)
{
    return wave_fold(v, [](N a, N b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v)
{
    return wave_fold(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    return wave_fold(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
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
    int64_t first_row, row_stride;  // first_row: of this launch
    int vocab, k;
    float factor;  // log2(e) / temperature
    double temperature;
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

constexpr int kRowParts = 8;  // of a thread's part of a row that is not kept

// A thread's sum of exponentials under its own largest logit so far.
template <typename T>
struct OnlineSum {
    typedef typename RowVec<T>::type vec;
    static constexpr int VE = RowShape<T>::VE;
    float top = -__builtin_inff(), sum = 0.0f;

    __device__ __forceinline__ float part(float z, float c, float mc) const { return exp2_fast(__builtin_fmaf(z, c, -mc)); }
    // `largest` of what comes next
    __device__ __forceinline__ void raise(float largest, float factor)
    {
        if (!(largest > top)) return;
        const float c = row_factor(largest, factor), mc = largest * c;
        sum = top == -__builtin_inff() ? sum : sum * exp2_fast(__builtin_fmaf(top, c, -mc));
        top = largest;
    }
    // The thread's whole part of a row; `parts`, one after another at a distance of BLOCK, are the largest of each of kRowParts runs of
    // `run` vectors.
    template <int BLOCK>
    __device__ __forceinline__ void add_row(const RowData<T, 0, BLOCK>& data, const RowShape<T>& s, float factor, int run, float* parts)
    {
        constexpr int kAhead = 4;  // vectors on their way at a time
        int v = threadIdx.x;
        for (int part = 0; part < kRowParts; ++part) {
            const int end = s.vectors < (part + 1) * run * BLOCK ? s.vectors : (part + 1) * run * BLOCK;
            float largest = -__builtin_inff();
            for (; v + (kAhead - 1) * BLOCK < end; v += kAhead * BLOCK) {
                raw_t x[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; ++j) x[j] = s.vector_at(v + j * BLOCK);
                largest = fmaxf(largest, add<kAhead>(x, factor));
            }
            for (; v < end; v += BLOCK) {
                const raw_t x[1] = {s.vector_at(v)};
                largest = fmaxf(largest, add<1>(x, factor));
            }
            parts[part * BLOCK] = largest;
        }
        if (data.lone_at >= 0) {
            const float z = to_float<T>(data.lone);
            raise(z, factor);
            add_element(z, factor);
        }
    }
    __device__ __forceinline__ void add_element(float z, float factor)
    {
        const float c = row_factor(top, factor);
        if (top != -__builtin_inff())
            sum += part(z, c, top * c);
        else if (z != z)  // among nothing but -inf so far, which adds nothing
            sum = z;
    }
    // (returns the largest of them)
    template <int N>
    __device__ __forceinline__ float add(const raw_t (&x)[N], float factor)
    {
        Largest<T> largest;
#pragma unroll
        for (int j = 0; j < N; ++j) largest.add(x[j]);
        raise(largest.get(), factor);
        const float c = row_factor(top, factor), mc = top * c;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const vec v = __builtin_bit_cast(vec, x[j]);
            if (top == -__builtin_inff()) {
#pragma unroll
                for (int e = 0; e < VE; ++e) add_element(to_float<T>(v[e]), factor);
                continue;
            }
            float all = 0.0f;
#pragma unroll
            for (int e = 0; e < VE; ++e) all += part(to_float<T>(v[e]), c, mc);
            sum += all;
        }
        return largest.get();
    }
    // the sum under the row's largest logit instead, whose factor is c
    __device__ __forceinline__ float under(float c, float mc) const
    {
        return top == -__builtin_inff() ? sum : sum * exp2_fast(__builtin_fmaf(top, c, -mc));
    }
};

__device__ __forceinline__ float number_of(uint32_t order)
{
    const uint32_t b = order & 0x80000000u ? order & 0x7FFFFFFFu : ~order;
    float x;
    __builtin_memcpy(&x, &b, 4);
    return x;  // (NaN: 0x7FFFFFFF)
}

constexpr int kBounds = 16;  // that are tried at a time

// Low bits of an order that say nothing: the type's own mantissa is shorter than fp32's by so many.
template <typename T>
constexpr int kLowBits = sizeof(T) == 4 ? 0 : __is_same(T, half_t) ? 13 : 16;

// What candidates are told apart and ordered by: order, then place, the lower first.
template <typename T>
__device__ __forceinline__ uint64_t entry_of(float x, int at)
{
    return (uint64_t)(order_of(x) >> kLowBits<T>) << 32 | (0xFFFFFFFFu - (uint32_t)at);
}

// The k largest entries of a row, whatever it holds, found bit by bit.  The row is read again for every bit: what it takes is no
// ordinary row's concern, and it needs no registers.  (n_found: 0 by now.)
template <typename T, int BLOCK>
__device__ __forceinline__ void keep_exactly(const T* row, int vocab, int k, uint64_t* found, int* n_found, int* counts)
{
    typedef typename RowVec<T>::type vec;
    constexpr int VE = RowShape<T>::VE;
    const RowShape<T> shape(row, vocab);
    RowData<T, 0, BLOCK> data;
    data.load(shape);
    __syncthreads();
    const int place_bits = 32 - __builtin_clz((uint32_t)vocab);
    uint64_t kth = 0;
    int turn = 0;
    for (int bit = 63 - kLowBits<T>; bit >= 0; --bit) {
        const uint64_t next = kth | 1ull << bit;
        if (bit < 32 && bit >= place_bits) {  // every entry has these
            kth = next;
            continue;
        }
        int count = 0;
        data.each(
            shape,
            [&](const vec& v, int i) PS_INLINE {
#pragma unroll
                for (int e = 0; e < VE; ++e) count += entry_of<T>(to_float<T>(v[e]), shape.element_of(i) + e) >= next;
            },
            [&](T x, int at) PS_INLINE { count += entry_of<T>(to_float<T>(x), at) >= next; });
        count = block_sum<BLOCK>(count, counts + turn * kBounds);
        turn ^= 1;
        if (count >= k) kth = next;
        if (count == k) break;
    }
    auto keep = [&](uint64_t entry) PS_INLINE {
        if (entry >= kth) found[atomicAdd(n_found, 1)] = entry;  // (k of them)
    };
    data.each(
        shape,
        [&](const vec& v, int i) PS_INLINE {
#pragma unroll
            for (int e = 0; e < VE; ++e) keep(entry_of<T>(to_float<T>(v[e]), shape.element_of(i) + e));
        },
        [&](T x, int at) PS_INLINE { keep(entry_of<T>(to_float<T>(x), at)); });
}

// 1. Every thread's largest element.  The k-th largest of these bounds the k-th largest of the row from below (k threads have one
//    at least as large), and few elements reach it: about k of them where k is small against the threads.  Any smaller bound does
//    too, so the search for it (kBounds at a time, each counted by a wave over all threads' largest) ends where little more than k
//    threads reach it.
// 2. Only those threads' vectors can hold candidates: the ones that do are handed over in LDS and spread over all threads.
// 3. A candidate's place is the number of larger ones.
// Where too many reach the bound (long runs of equal logits), or NaN or infinities are in the row, keep_exactly finds the k-th largest
// (order, place) bit by bit: all are different, so exactly k reach it.
// Of 155 us for 8192 x 50257, reading and the sum are 132; the search 10, the vectors 15 to 24, the elements 20, the places 17 (each alone,
// partly hidden).  Tried: candidates read again from memory (50 us more), a vector's elements one after another by one thread (40
// more), one wave for all places (25 more), workgroups that have the next row on its way (30 more: they fill the registers).
template <typename T, int NV, int BLOCK>
__global__ __launch_bounds__(BLOCK, BLOCK == 512 && NV <= 14 ? 6 : 4) void top_logits_kernel(TopArgs p)
{
    typedef typename RowVec<T>::type vec;
    constexpr int VE = RowShape<T>::VE;
    constexpr int kWaves = BLOCK / 64, kPerWave = kBounds / kWaves;  // (BLOCK <= 1024)
    constexpr int kTopCandidates = BLOCK == 256 ? 512 : 2048;
    constexpr int kSlots = NV == 0 ? 2048 : BLOCK == 256 ? 256 : 1024;
    __shared__ uint64_t found[kTopCandidates];
    __shared__ raw_t slots[NV > 0 ? kSlots : 1];  // vectors that hold candidates
    __shared__ int slot_vector[kSlots];           // their numbers (of a row that is not kept: the first one's of a run)
    __shared__ float part_largest[NV > 0 ? 1 : kRowParts * BLOCK];
    __shared__ uint32_t largest[BLOCK];
    __shared__ int place_of[BLOCK];
    __shared__ uint32_t lds_max[kWaves], lds_min[kWaves];
    __shared__ float lds_sum[kWaves];
    __shared__ int lds_count[2][kBounds];  // (as many as waves, at least)
    __shared__ int n_found, n_slots;
    const int thread = threadIdx.x, lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int64_t r = p.first_row + blockIdx.x;
    const T* row = static_cast<const T*>(p.logits) + r * p.row_stride;
    const RowShape<T> shape(row, p.vocab);
    RowData<T, NV, BLOCK> data;
    data.load(shape);
    // A row that is not kept is read once for both: a thread's sum goes by its own largest so far.  Of every thread's part it is kept where
    // its large elements are.
    const int each = (shape.vectors + BLOCK - 1) / BLOCK, run = (each + kRowParts - 1) / kRowParts;  // vectors of a thread, of a run of its
    OnlineSum<T> online;
    float my_top;
    if constexpr (NV == 0) {
        online.add_row(data, shape, p.factor, run, part_largest + thread);
        my_top = online.top;
    } else {
        my_top = data.largest(shape);
    }
    const uint32_t mine = order_of(my_top);  // (of a thread without elements: -inf's)
    largest[thread] = mine;
    if (thread == 0) n_found = n_slots = 0;
    {
        const uint32_t hi = wave_max(mine), lo = ~wave_max(~mine);
        if (lane == 0) lds_max[wave] = hi, lds_min[wave] = lo;
    }
    __syncthreads();
    uint32_t most = lds_max[0], least = lds_min[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        most = lds_max[w] > most ? lds_max[w] : most;
        least = lds_min[w] < least ? lds_min[w] : least;
    }
    const float m = number_of(most), c = row_factor(m, p.factor), mc = m * c;
    // the sum of exponentials; NaN where a logit is NaN or infinite
    float sum = 0.0f;
    if (NV == 0) {
        sum = online.under(c, mc);
    } else {
        data.hide();
        data.each(
            shape,
            [&](const vec& v, int) PS_INLINE {
                float part = 0.0f;
#pragma unroll
                for (int e = 0; e < VE; ++e) part += exp2_fast(__builtin_fmaf(to_float<T>(v[e]), c, -mc));
                sum += part;
            },
            [&](T x, int) PS_INLINE { sum += exp2_fast(__builtin_fmaf(to_float<T>(x), c, -mc)); });
    }
    sum = wave_sum(sum);
    if (lane == 0) lds_sum[wave] = sum;
    // the bound: at least k threads reach `bound`, fewer than k `above`
    uint32_t bound = least, above = most + (most != 0xFFFFFFFFu);
    int reach = BLOCK;
    if (p.k <= BLOCK) {
        const int enough = p.k + p.k / 4 + 8;
        int turn = 0;
        uint32_t others[kWaves];
#pragma unroll
        for (int j = 0; j < kWaves; ++j) others[j] = largest[j * 64 + lane];
        while (reach > enough && above - bound > 1) {
            const uint32_t step = (above - bound) / (kBounds + 1), left = (above - bound) % (kBounds + 1);
            auto tried = [&](uint32_t i) PS_INLINE { return bound + step * (i + 1) + (left * (i + 1)) / (kBounds + 1); };
#pragma unroll
            for (int i = 0; i < kPerWave; ++i) {
                const uint32_t limit = tried(wave * kPerWave + i);
                int n = 0;
#pragma unroll
                for (int j = 0; j < kWaves; ++j) n += __popcll(__ballot(others[j] >= limit));
                if (lane == 0) lds_count[turn][wave * kPerWave + i] = n;
            }
            __syncthreads();
            // the bounds rise, so the ones that k threads reach are the first of them
            const int count = lds_count[turn][lane & (kBounds - 1)];
            const int reached = __popcll(__ballot(count >= p.k) & ((1u << kBounds) - 1));
            const uint32_t new_bound = reached > 0 ? tried(reached - 1) : bound;
            if (reached < kBounds) above = tried(reached);
            if (reached > 0) reach = __builtin_amdgcn_readlane(count, reached - 1);
            bound = new_bound;
            turn ^= 1;
        }
    }
    __syncthreads();
    sum = lds_sum[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += lds_sum[w];
    const bool ordinary = sum - sum == 0.0f;
    auto value_of = [](uint64_t entry) PS_INLINE {
        const uint32_t order = (uint32_t)(entry >> 32) << kLowBits<T>;
        return number_of(order & 0x80000000u ? order : order | ((1u << kLowBits<T>) - 1));
    };
    auto keep = [&](uint64_t entry) PS_INLINE {
        const int at = atomicAdd(&n_found, 1);
        if (at < kTopCandidates) found[at] = entry;
    };
    // the elements of a vector that reach the limit: one addition for all of them
    const float limit = number_of(bound);
    auto keep_of = [&](const vec& x, int first) PS_INLINE {
        uint32_t reaches = 0;
#pragma unroll
        for (int e = 0; e < VE; ++e) reaches |= to_float<T>(x[e]) >= limit ? 1u << e : 0u;
        if (!reaches) return;
        int at = atomicAdd(&n_found, __popc(reaches));
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            if (!(reaches >> e & 1)) continue;
            if (at < kTopCandidates) found[at] = entry_of<T>(to_float<T>(x[e]), first + e);
            ++at;
        }
    };
    bool few = ordinary && p.k <= BLOCK && reach <= 2 * p.k + 64;
    if (few && NV > 0) {
        // a thread that reaches the bound leaves those of its vectors that do
        if (mine >= bound) {
            uint32_t reaches = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                Largest<T> top;
                top.add(data.kept[i]);
                if (i * BLOCK + thread < shape.vectors && top.get() >= limit) reaches |= 1u << i;
            }
            if (reaches) {
                int at = atomicAdd(&n_slots, __popc(reaches));
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (!(reaches >> i & 1)) continue;
                    if (at < kSlots) slots[at] = data.kept[i], slot_vector[at] = i * BLOCK + thread;
                    ++at;
                }
            }
            if (data.lone_at >= 0 && to_float<T>(data.lone) >= limit) keep(entry_of<T>(to_float<T>(data.lone), data.lone_at));
        }
        __syncthreads();
        const int n = n_slots;
        few = n <= kSlots;
        // an element a thread, and one addition a wave
        const T* elements = reinterpret_cast<const T*>(slots);
        for (int first = wave * 64; few && first < n * VE; first += BLOCK) {
            const int i = first + lane;
            const float x = i < n * VE ? to_float<T>(elements[i]) : 0.0f;
            const bool reaches = i < n * VE && x >= limit;
            const uint64_t all = __ballot(reaches);
            int at = 0;
            if (lane == 0 && all) at = atomicAdd(&n_found, __popcll(all));
            at = __builtin_amdgcn_readfirstlane(at) + __popcll(all & ((1ull << lane) - 1));
            if (reaches && at < kTopCandidates) found[at] = entry_of<T>(x, shape.element_of(slot_vector[i / VE]) + i % VE);
        }
        __syncthreads();
        few = few && n_found <= kTopCandidates;
    } else if (few) {
        // of a row that is not kept, the runs that reach the bound are read again, spread over all threads
        if (mine >= bound) {
            uint32_t reaches = 0;
#pragma unroll
            for (int i = 0; i < kRowParts; ++i) reaches |= part_largest[i * BLOCK + thread] >= limit ? 1u << i : 0u;
            if (reaches) {
                int at = atomicAdd(&n_slots, __popc(reaches));
                for (int i = 0; i < kRowParts; ++i)
                    if (reaches >> i & 1) {
                        if (at < kSlots) slot_vector[at] = i * run * BLOCK + thread;
                        ++at;
                    }
            }
            if (data.lone_at >= 0 && to_float<T>(data.lone) >= limit) keep(entry_of<T>(to_float<T>(data.lone), data.lone_at));
        }
        __syncthreads();
        few = n_slots <= kSlots;
        const int items = few ? n_slots * run : 0;
        constexpr int kAhead = 4;  // vectors on their way at a time
        for (int first = thread; first < items; first += kAhead * BLOCK) {
            raw_t x[kAhead];
            int v[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int i = first + j * BLOCK, slot = i / run;
                v[j] = i < items ? (i - slot * run) * BLOCK + slot_vector[slot] : shape.vectors;
                asm volatile("" : "=v"(x[j]));
                if (v[j] < shape.vectors) x[j] = shape.vector_at(v[j]);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (v[j] < shape.vectors) keep_of(__builtin_bit_cast(vec, x[j]), shape.element_of(v[j]));
        }
        __syncthreads();
        few = few && n_found <= kTopCandidates;
    }
    if (!few) {
        __syncthreads();  // everyone has seen how many there were
        if (thread == 0) n_found = 0;
        keep_exactly<T, BLOCK>(row, p.vocab, p.k, found, &n_found, lds_count[0]);
        __syncthreads();
    }
    const int n = n_found;
    if (thread == 0) {
        float lse = (float)log_sum(m, __builtin_fmaf(m, c, -mc), (double)sum, p.temperature);
        if (!ordinary) {  // the row's largest, NaN being larger than everything: a row of -inf alone has no mass
            uint64_t first = 0;
            for (int i = 0; i < n; ++i) first = found[i] > first ? found[i] : first;
            lse = (uint32_t)(first >> 32) == 0xFFFFFFFFu >> kLowBits<T> ? __builtin_nanf("") : value_of(first);
        }
        *global(p.lse + r) = lse;
    }
    auto write = [&](uint64_t entry, int place) PS_INLINE {
        const uint32_t at = 0xFFFFFFFFu - (uint32_t)entry;
        const float x = value_of(entry);
        T value = from_float<T>(x);
        if (!(x < 0.0f || x > 0.0f)) value = *global(row + at);  // a zero's sign, a NaN's bits
        *global(p.ids + r * p.k + place) = (int32_t)at;
        *global(static_cast<T*>(p.values) + r * p.k + place) = value;
    };
    if (n <= BLOCK) {
        int span = 64;
        while (span < n) span *= 2;
        const int slices = BLOCK / span, mine_at = thread & (span - 1), slice = thread / span;
        place_of[thread] = 0;
        __syncthreads();
        const uint64_t entry = mine_at < n ? found[mine_at] : 0;
        int count = 0;
#pragma unroll 4
        for (int j = slice; j < n; j += slices) count += found[j] > entry;
        if (mine_at < n && count) atomicAdd(&place_of[mine_at], count);
        __syncthreads();
        const int place = place_of[mine_at];
        if (slice == 0 && mine_at < n && place < p.k) write(entry, place);
    } else {
        for (int i = thread; i < n; i += BLOCK) {
            const uint64_t entry = found[i];
            int place = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) place += found[j] > entry;
            if (place < p.k) write(entry, place);
        }
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
    float* denominator;   // rows that count: made here (count_rows), or before; nullptr: `count`
    void* grad;
    const float* upstream;
    float* upstream_used;
    int64_t rows, first_row, row_stride, ids_stride, values_stride, upstream_stride;  // first_row: of this launch
    int64_t ignore_index;
    int vocab, k;
    int values_dtype;
    float factor, factor_low;  // log2(e) / temperature is their sum
    float temperature_f, label_weight, upstream_value, count;
    double temperature, inv_temperature;
    bool ids_64, labels_64;
    bool count_rows;      // few enough for every workgroup to count them itself
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

// How the two softmaxes of a row, at the temperature and at 1, come from one another: at temperature 1, or if only one of the two is
// wanted, there is one; at 2 the second's exponential is the first's square; else each has its own.
enum { kOne, kSquare, kTwo };

// Calls f(Int<how>) for the row's way.
template <typename F>
__device__ __forceinline__ auto with_softmaxes(const DistillArgs& p, F f)
{
    const bool both = p.label_weight != 0.0f && p.label_weight != 1.0f;
    if (!both || p.temperature == 1.0) return f(Int<kOne>());
    if (p.temperature == 2.0) return f(Int<kSquare>());
    return f(Int<kTwo>());
}

// The exponentials of a logit: e at the temperature (at 1 if there is no other), e1 at 1.  Of fp32 logits the factor is taken in two
// parts: its rounding, 2^-25 of every exponent, is more than their own.
struct Exponents {
    float c, c_low, mc, c1, c1_low, mc1;

    __device__ __forceinline__ Exponents(const DistillArgs& p, float m)
    {
        constexpr float kLog2eLow = 1.9259630e-8f;  // log2(e) = kLog2e + this
        const float own = p.label_weight == 1.0f ? kLog2e : p.factor, own_low = p.label_weight == 1.0f ? kLog2eLow : p.factor_low;
        c = row_factor(m, own);
        c_low = c == own ? own_low : 0.0f;
        mc = m * c;
        c1 = row_factor(m, kLog2e);
        c1_low = c1 == kLog2e ? kLog2eLow : 0.0f;
        mc1 = m * c1;
    }
    template <int HOW, bool LOW>
    __device__ __forceinline__ void of(float z, float& e, float& e1) const
    {
        e = exp2_fast(__builtin_fmaf(z, c, LOW ? __builtin_fmaf(z, c_low, -mc) : -mc));
        if (HOW == kOne) e1 = e;
        if (HOW == kSquare) e1 = e * e;
        if (HOW == kTwo) e1 = exp2_fast(__builtin_fmaf(z, c1, LOW ? __builtin_fmaf(z, c1_low, -mc1) : -mc1));
    }
    // what exp2(-.) brings sums of e, or e1, to sums of exp((z - m) / temperature)
    template <bool LOW>
    __device__ __forceinline__ float bias(float m) const
    {
        return __builtin_fmaf(m, c, LOW ? __builtin_fmaf(m, c_low, -mc) : -mc);
    }
    template <bool LOW>
    __device__ __forceinline__ float bias1(float m) const
    {
        return __builtin_fmaf(m, c1, LOW ? __builtin_fmaf(m, c1_low, -mc1) : -mc1);
    }
};

// The teacher's list in LDS: ids, probabilities and, if wanted, by how much an entry's logit is above the student's, over the
// temperature.  `mass`: the probabilities' sum.  Their logarithms are value / temperature less `base` and less log(`norm`).  Where the rest
// counts, 1 - mass does, and of a student near its teacher nothing but the difference of such numbers is left: for fp32 logits they are
// made in 64 bits.  (16-bit logits are known to 2^-9 or 2^-12 themselves, and the registers that it takes are a workgroup less on a
// CU: the loss of 4096 x 30522 took 72 us instead of 54.)
template <typename T>
using ListSum = std::conditional_t<sizeof(T) == 4, double, float>;

template <int BLOCK, typename T>
__device__ __forceinline__ void load_list(const DistillArgs& p, int64_t r, const RowShape<T>& shape, int* ids, float* prob, float* above, float* lds_a,
                                          ListSum<T>* lds_b, ListSum<T>& mass, float& base, ListSum<T>& norm)
{
    const bool rest = p.teacher_lse != nullptr;
    const float given = rest ? *global(p.teacher_lse + r) : 0.0f;
    float top = -__builtin_inff();
    ListSum<T> sum = 0;
    for (int i = threadIdx.x; i < p.k; i += BLOCK) {
        const int64_t id = whole_at(p.ids, r * p.ids_stride + i, p.ids_64);
        const float value = value_at(p.values, r * p.values_stride + i, p.values_dtype);
        ids[i] = id < 0 ? -1 : id < p.vocab ? (int)id : -2;  // -2: beyond the vocabulary
        prob[i] = value / p.temperature_f;
        if (above) above[i] = ids[i] >= 0 ? (value - to_float<T>(*global(shape.row + id))) / p.temperature_f : 0.0f;
        if (id >= 0) top = fmaxf(top, prob[i]);
        if (rest) {
            ListSum<T> e = 0;
            if (id >= 0) {
                if constexpr (sizeof(T) == 4)
                    e = exp((double)value * p.inv_temperature - (double)given);
                else
                    e = expf(prob[i] - given);
            }
            prob[i] = (float)e;
            sum += e;
        }
    }
    if (!rest) {
        top = block_max<BLOCK, float>(top, lds_a);
        for (int i = threadIdx.x; i < p.k; i += BLOCK) {  // (a thread's own entries)
            const float e = ids[i] == -1 ? 0.0f : expf(prob[i] - top);
            prob[i] = e;
            sum += e;
        }
    }
    mass = block_sum<BLOCK>(sum, lds_b);
    base = rest ? given : top;
    norm = 1;
    if (!rest) {
        norm = mass;
        const float scale = mass > 0 ? 1.0f / (float)mass : mass == mass ? 0.0f : (float)mass;
        for (int i = threadIdx.x; i < p.k; i += BLOCK) prob[i] *= scale;
        mass = mass > 0 ? 1 : mass;
    }
    __syncthreads();
}

// The row's gradient, from registers or memory: list entries and label after everything else, over it.
template <typename T, int NV, int BLOCK>
__device__ __forceinline__ void write_gradient(const DistillArgs& p, int64_t r, const RowShape<T>& shape, RowData<T, NV, BLOCK>& data,
                                               const RowStats& s, float factor, const int* ids, const float* prob, int64_t label)
{
    typedef typename RowVec<T>::type vec;
    constexpr int VE = RowShape<T>::VE;
    T* out = static_cast<T*>(p.grad) + r * (int64_t)p.vocab;
    const bool soft_there = p.label_weight != 1.0f, hard_there = p.label_weight != 0.0f;
    const float soft = soft_there ? factor * (1.0f - p.label_weight) * p.temperature_f * s.inv_s : 0.0f;
    const float hard = hard_there ? factor * p.label_weight * s.inv_s1 : 0.0f;
    const float off = soft_there ? soft * s.coef : 0.0f;
    const Exponents exponents(p, s.m);
    data.hide();
    with_softmaxes(p, [&](auto how) PS_INLINE {
        const float share = how() == kOne ? off + hard : off;
        auto gradient = [&](float z) PS_INLINE {
            float e, e1;
            exponents.of<how(), sizeof(T) == 4>(z, e, e1);
            return __builtin_fmaf(e, share, how() == kOne ? 0.0f : e1 * hard);
        };
        data.each(
            shape,
            [&](const vec& v, int i) PS_INLINE {
                vec g;
#pragma unroll
                for (int e = 0; e < VE; ++e) g[e] = from_float<T>(gradient(to_float<T>(v[e])));
                shape.store(out, i, g);
            },
            [&](T x, int at) PS_INLINE { *global(out + at) = from_float<T>(gradient(to_float<T>(x))); });
        __syncthreads();
        const float mass_share = p.teacher_lse != nullptr ? soft : off;
        const float given = factor * (1.0f - p.label_weight) * p.temperature_f;
        if (soft_there) {
            for (int i = threadIdx.x; i < p.k; i += BLOCK) {
                const int id = ids[i];
                if (id < 0) continue;
                float e, e1;
                exponents.of<how(), sizeof(T) == 4>(to_float<T>(*global(shape.row + id)), e, e1);
                float g = __builtin_fmaf(e, mass_share, -given * prob[i]);
                if (hard_there) g += e1 * hard - (id == label ? factor * p.label_weight : 0.0f);
                *global(out + id) = from_float<T>(g);
            }
        }
        if (hard_there) {
            // the label, unless it is on the list: the thread of its entry has written it
            bool listed = false;
            if (soft_there)
                for (int i = threadIdx.x; i < p.k; i += BLOCK) listed |= ids[i] == label;
            if (!__syncthreads_or(listed) && threadIdx.x == 0 && label >= 0 && label < p.vocab)
                *global(out + label) = from_float<T>(gradient(to_float<T>(*global(shape.row + label))) - factor * p.label_weight);
        }
    });
}

template <typename T, int NV, int BLOCK>
__device__ __forceinline__ void write_zeros(const DistillArgs& p, int64_t r, const RowShape<T>& shape)
{
    typedef typename RowVec<T>::type vec;
    T* out = static_cast<T*>(p.grad) + r * (int64_t)p.vocab;
    vec zero;
#pragma unroll
    for (int e = 0; e < RowShape<T>::VE; ++e) zero[e] = (T)0.0f;
    for (int v = threadIdx.x; v < shape.vectors; v += BLOCK) shape.store(out, v, zero);
    const int lone = shape.lone_of(threadIdx.x);
    if (lone >= 0) *global(out + lone) = (T)0.0f;
}

// Words of LDS that hold a bit for every token.  The first token's bit is moved so that a vector's bits begin at its own byte or half
// byte.
__host__ __device__ constexpr int member_words(int vocab) { return (vocab + 8 + 31) / 32; }

template <typename T>
struct Members {
    static constexpr int VE = RowShape<T>::VE;
    uint32_t* words;
    int shift;

    __device__ __forceinline__ Members(uint32_t* w, const RowShape<T>& s) : words(w), shift((VE - s.head) & (VE - 1)) {}
    // whether it was there
    __device__ __forceinline__ bool add(int id) const
    {
        const int bit = id + shift;
        return atomicOr(&words[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1;
    }
    __device__ __forceinline__ bool has(int id) const { return words[(id + shift) >> 5] >> ((id + shift) & 31) & 1; }
    // the bits of the vector that begins with this element
    __device__ __forceinline__ uint32_t of_vector(int first) const
    {
        const uint32_t bit = (uint32_t)(first + shift);
        return reinterpret_cast<const uint8_t*>(words)[bit >> 3] >> (bit & 7) & ((1u << VE) - 1);
    }
};

struct RowSums {
    float all, rest, at_1;  // of the exponentials: everything, off the list, at temperature 1
};

// A thread's part of the row's sums.
template <int HOW, bool REST, typename T, int NV, int BLOCK>
__device__ __forceinline__ RowSums add_up(const RowData<T, NV, BLOCK>& data, const RowShape<T>& shape, const Exponents& exponents,
                                          const Members<T>& members)
{
    constexpr int VE = RowShape<T>::VE;
    float all = 0.0f, rest = 0.0f, at_1 = 0.0f;
    data.each(
        shape,
        [&](const typename RowVec<T>::type& v, int i) PS_INLINE {
            float part = 0.0f;
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                float e, e1;
                exponents.of<HOW, sizeof(T) == 4>(to_float<T>(v[k]), e, e1);
                part += e;
                if (HOW != kOne) at_1 += e1;
            }
            all += part;
            if (REST) rest += members.of_vector(shape.element_of(i)) ? 0.0f : part;
        },
        [&](T z, int at) PS_INLINE {
            float e, e1;
            exponents.of<HOW, sizeof(T) == 4>(to_float<T>(z), e, e1);
            all += e;
            if (HOW != kOne) at_1 += e1;
            if (REST && !members.has(at)) rest += e;
        });
    return {all, rest, HOW == kOne ? all : at_1};
}

// Loss, and the gradient in the same pass over the row: maximum, sums, then exponentials again from the registers (keeping them would
// take twice the registers).  At the speed of a copy of the rows; the list's part (k entries, 64-bit logarithms on a lane each) runs
// beside other workgroups' reads.  The gradient's vectors start where the logits' do, at any element of an output row.
// Dynamic LDS: a bit for every token of the vocabulary (is it on the list?), then the list's ids and probabilities.
template <typename T, int NV, int BLOCK>
__global__ __launch_bounds__(BLOCK, 4) void distill_loss_kernel(DistillArgs p)
{
    typedef typename RowVec<T>::type vec;
    constexpr int VE = RowShape<T>::VE;
    extern __shared__ uint32_t dynamic[];
    __shared__ float lds[6][BLOCK / 64];
    __shared__ ListSum<T> lds_list[2][BLOCK / 64];
    const int words = member_words(p.vocab);
    uint32_t* member = dynamic;
    int* ids = reinterpret_cast<int*>(dynamic + words);
    float* prob = reinterpret_cast<float*>(dynamic + words + p.k);
    float* above = prob + p.k;
    const bool rest = p.teacher_lse != nullptr;
    const bool soft = p.label_weight != 1.0f, hard = p.label_weight != 0.0f;
    const float upstream = p.upstream ? *global(p.upstream) : p.upstream_value;
    if (p.upstream_used && p.first_row + blockIdx.x == 0 && threadIdx.x == 0) *global(p.upstream_used) = upstream;
    float count = p.denominator && !p.count_rows ? *global(p.denominator) : p.count;
    if (p.count_rows) {
        int n = 0;
        for (int i = threadIdx.x; i < (int)p.rows; i += BLOCK) n += whole_at(p.labels, i, p.labels_64) != p.ignore_index;
        n = block_sum<BLOCK>(n, reinterpret_cast<int*>(lds[5]));
        count = (float)(n > 0 ? n : 1);
        if (p.first_row + blockIdx.x == 0 && threadIdx.x == 0) *global(p.denominator) = count;
    }
    const float inv_count = 1.0f / count;
    const int64_t r = p.first_row + blockIdx.x;
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
            return;
        }
        if (hard) wrong = label < 0 || label >= p.vocab;
    }
    RowData<T, NV, BLOCK> data;
    data.load(shape);
    for (int i = threadIdx.x; i < words; i += BLOCK) member[i] = 0;
    ListSum<T> mass, norm;
    float base;
    load_list<BLOCK>(p, r, shape, ids, prob, above, lds[0], lds_list[0], mass, base, norm);
    const Members<T> members(member, shape);
    for (int i = threadIdx.x; i < p.k; i += BLOCK) {
        const int id = ids[i];
        wrong |= id >= 0 ? members.add(id) : id == -2;
    }
    const float m = block_max<BLOCK, float>(data.largest(shape), lds[2]);  // (a barrier: the members are there)
    const Exponents exponents(p, m);
    data.hide();
    const RowSums sums = with_softmaxes(p, [&](auto how) PS_INLINE {
        if (rest && soft) return add_up<how(), true, T, NV, BLOCK>(data, shape, exponents, members);
        return add_up<how(), false, T, NV, BLOCK>(data, shape, exponents, members);
    });
    float sum = sums.all, sum_rest = sums.rest, sum1 = sums.at_1;
    if (rest && soft) {
        // what is off the list in vectors that hold a token of it: the thread of the first such token sees to it
        for (int i = threadIdx.x; i < p.k; i += BLOCK) {
            const int id = ids[i];
            if (id < shape.head || id >= shape.element_of(shape.vectors)) continue;
            const int number = (id - shape.head) / VE, first = shape.element_of(number);
            const uint32_t bits = members.of_vector(first);
            if (bits & ((1u << (id - first)) - 1)) continue;
            const vec v = __builtin_bit_cast(vec, shape.vector_at(number));
            const auto off_list = [&](float z) PS_INLINE {
                float x, x1;
                exponents.of<kOne, sizeof(T) == 4>(z, x, x1);
                return x;
            };
#pragma unroll
            for (int e = 0; e < VE; ++e)
                sum_rest += bits >> e & 1 ? 0.0f : off_list(to_float<T>(v[e]));
        }
    }
    // The list's part of the divergence: sum p (log p - log q), the two logarithms being value / temperature and z / temperature, each
    // less its log-sum-exp.  The large ones never meet: sums of the differences here, the difference of the sums below.
    // With the rest, an fp32 student's sum is that off the list and the list's own, the latter in 64 bits like the teacher's: an error of
    // the former then counts by how far the two rests are apart, not by itself.
    float term = 0.0f;
    ListSum<T> sum_list = 0;
    if (soft) {
        for (int i = threadIdx.x; i < p.k; i += BLOCK) {
            if (ids[i] < 0) continue;
            if (prob[i] != 0.0f) term = __builtin_fmaf(prob[i], above[i], term);
            if (rest && sizeof(T) == 4) sum_list += exp(((double)to_float<T>(*global(shape.row + ids[i])) - (double)m) * p.inv_temperature);
        }
    }
    if (rest && soft && sizeof(T) == 4) sum_list = block_sum<BLOCK>(sum_list, lds_list[1]);
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
    if (wrong) sum = sum1 = __builtin_nanf("");
    RowStats s;
    s.m = m;
    s.inv_s = 1.0f / sum;
    s.inv_s1 = 1.0f / sum1;
    const ListSum<T> p_rest = rest && mass < 1 ? 1 - mass : 0;
    const double bias = 0.6931471805599453 * (double)exponents.bias<sizeof(T) == 4>(m);
    ListSum<T> off_list = sum_rest, everything = sum;  // (of 16-bit logits: both with the bias)
    if constexpr (sizeof(T) == 4) {
        off_list = (double)sum_rest * (1.0 - bias * (1.0 - 0.5 * bias));  // (a rounding's, far below 1: to the second order)
        everything = off_list + sum_list;
    }
    s.coef = rest ? (p_rest == 0 ? 1.0f : (float)(off_list - p_rest * everything) / (float)off_list) : (float)mass;
    if (threadIdx.x < 64) {
        // the row's logarithms, a lane each
        const int lane = threadIdx.x;
        const bool biased = !rest || sizeof(T) == 2;
        const double z_sum = biased ? (double)sum : (double)everything;
        const double argument = lane == 0 ? z_sum : lane == 1 ? (double)norm : lane == 2 ? (double)p_rest : lane == 3 ? (double)off_list : lane == 4 ? (double)sum1 : 1.0;
        const double logarithm = log(argument);
        const double log_z = of_lane(logarithm, 0), log_norm = of_lane(logarithm, 1), log_p = of_lane(logarithm, 2);
        const double log_off = of_lane(logarithm, 3), log_1 = of_lane(logarithm, 4);
        if (lane == 0) {
            double loss = 0.0;
            if (soft) {
                double kl = (double)term;
                if (mass != 0) {
                    const double lse = (double)m * p.inv_temperature + log_z - (biased ? bias : 0.0);
                    kl += (double)mass * (lse - (double)base - log_norm);
                }
                if (p_rest > 0) kl += (double)p_rest * (log_p + log_z - log_off);
                if (wrong) kl = __builtin_nan("");
                loss = (1.0 - (double)p.label_weight) * p.temperature * p.temperature * kl;
            }
            if (hard) {
                const float z = wrong ? m : to_float<T>(*global(shape.row + label));
                loss += (double)p.label_weight * ((double)m + log_1 - 0.6931471805599453 * (double)exponents.bias1<sizeof(T) == 4>(m) - (double)z);
            }
            *global(p.row_loss + r) = (float)loss;
            if (p.stats) {
                *global(p.stats + 4 * r) = s.m;
                *global(p.stats + 4 * r + 1) = s.inv_s;
                *global(p.stats + 4 * r + 2) = s.coef;
                *global(p.stats + 4 * r + 3) = s.inv_s1;
            }
        }
    }
    if (p.grad) write_gradient<T, NV, BLOCK>(p, r, shape, data, s, upstream * inv_count, ids, prob, label);
}

// The gradient from the row's stats: one read, one write.  Where the forward pass has made it, a launch of workgroups that end (4 us).
template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void distill_backward_kernel(DistillArgs p)
{
    extern __shared__ uint32_t dynamic[];
    __shared__ float lds[BLOCK / 64];
    __shared__ ListSum<T> lds_list[BLOCK / 64];
    // the gradient that the forward pass made is at this very factor
    if (p.upstream_used && *global(p.upstream) == *global(p.upstream_used)) return;
    int* ids = reinterpret_cast<int*>(dynamic);
    float* prob = reinterpret_cast<float*>(dynamic + p.k);
    const float inv_count = 1.0f / (p.denominator ? *global(p.denominator) : p.count);
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
        ListSum<T> mass, norm;
        float base;
        load_list<BLOCK, T>(p, r, shape, ids, prob, nullptr, lds, lds_list, mass, base, norm);
        RowData<T, 0, BLOCK> data;
        data.load(shape);
        write_gradient<T, 0, BLOCK>(p, r, shape, data, s, *global(p.upstream + r * p.upstream_stride) * inv_count, ids, prob, label);
        __syncthreads();  // before the next row's list
    }
}

// One workgroup: how many rows count (at least 1).
__global__ __launch_bounds__(1024) void count_rows_kernel(const void* labels, bool is64, int64_t rows, int64_t ignore_index, float* out)
{
    __shared__ int lds[16];
    int n = 0;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) n += whole_at(labels, r, is64) != ignore_index;
    n = block_sum<1024>(n, lds);
    if (threadIdx.x == 0) *global(out) = (float)(n > 0 ? n : 1);
}

// One workgroup, a fixed order: the same rows give the same loss.  In 64 bits: a row more costs nothing here.
__global__ __launch_bounds__(1024) void sum_rows_kernel(const float* row_loss, int64_t rows, const float* denominator, float count, float* out)
{
    __shared__ double lds[1024];
    double sum = 0.0;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) sum += (double)*global(row_loss + r);
    lds[threadIdx.x] = sum;
    for (int n = 512; n; n >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < n) lds[threadIdx.x] += lds[threadIdx.x + n];
    }
    if (threadIdx.x == 0) *global(out) = (float)(lds[0] / (double)(denominator ? *global(denominator) : count));
}

}  // namespace

#endif  // PS_LOGITS_H
