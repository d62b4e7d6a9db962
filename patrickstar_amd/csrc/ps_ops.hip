// The C ABI of include/ps_ops.h: checks of the descriptors, launch shapes, launches.  Kernels: ps_rotary.h, ps_logits.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "ps_ops.h"

#include "ps_error.h"
#include "ps_rotary.h"
#include "ps_logits.h"

namespace {

constexpr int kCus = 256;

// Workgroups of the rotations, which loop over their tokens.
constexpr uint32_t kForwardBlocks = 64 * kCus, kBackwardBlocks = 4 * kCus;
constexpr int64_t kCachedBytes = 32 << 20;  // outputs up to so long are written through the L2 caches for whoever reads them next

int size_of(int dtype) { return dtype == PS_F32 ? 4 : 2; }

bool known(int dtype) { return dtype == PS_F16 || dtype == PS_BF16 || dtype == PS_F32; }

// Calls f(a value of the element type).
template <typename F>
void with_type(int dtype, F f)
{
    if (dtype == PS_F16)
        f(half_t());
    else if (dtype == PS_BF16)
        f(bf16_t());
    else
        f(float());
}

// ---------------------------------------------------------------------------------------------------------- rotations

int check_heads(const ps_heads_call* c, bool backward)
{
    if (!c) return fail(PS_ERR_BAD_ARG, "call is NULL");
    if (!known(c->dtype)) return fail(PS_ERR_BAD_ARG, "dtype %d is unknown", c->dtype);
    if (c->weight_dtype != c->dtype && c->weight_dtype != PS_F32)
        return fail(PS_ERR_BAD_ARG, "weight_dtype %d: the elements' own type or PS_F32", c->weight_dtype);
    if (c->position_bytes != 4 && c->position_bytes != 8) return fail(PS_ERR_BAD_ARG, "position_bytes = %d", c->position_bytes);
    if (c->dim < 1 || c->dim > PS_MAX_HEAD_DIM) return fail(PS_ERR_BAD_ARG, "dim = %d is not in 1 .. %d", c->dim, PS_MAX_HEAD_DIM);
    if (c->rotary < 0 || c->rotary % 2 || c->rotary > c->dim)
        return fail(PS_ERR_BAD_ARG, "rotary = %d must be even and at most dim = %d", c->rotary, c->dim);
    if (c->axes < 1) return fail(PS_ERR_BAD_ARG, "axes = %d", c->axes);
    if (c->batch < 0 || c->tokens < 0 || c->heads[0] < 0 || c->heads[1] < 0) return fail(PS_ERR_BAD_ARG, "a negative size");
    if (c->heads[0] > (1 << 20) || c->heads[1] > (1 << 20)) return fail(PS_ERR_BAD_ARG, "more than 2^20 heads");
    if (c->tokens && c->batch > INT32_MAX / c->tokens) return fail(PS_ERR_BAD_ARG, "more than 2^31 - 1 tokens");
    if (!(c->eps >= 0.0f)) return fail(PS_ERR_BAD_ARG, "eps = %g", (double)c->eps);
    if (c->batch * c->tokens == 0) return 0;
    for (int w = 0; w < 2; ++w) {
        if (c->heads[w] == 0) continue;
        if (!c->x[w] || !c->out[w] || (backward && !c->grad[w])) return fail(PS_ERR_BAD_ARG, "%s have a NULL address", w ? "keys" : "queries");
        const uintptr_t bytes = (uintptr_t)size_of(c->dtype);
        if ((uintptr_t)c->x[w] % bytes || (uintptr_t)c->out[w] % bytes || (backward && (uintptr_t)c->grad[w] % bytes))
            return fail(PS_ERR_BAD_ARG, "%s are not aligned to their type", w ? "keys" : "queries");
        if (c->weight_grad[w] && !c->weight[w]) return fail(PS_ERR_BAD_ARG, "a gradient is wanted of a weight that is not there");
    }
    if (c->rotary && (!c->positions || !c->plan)) return fail(PS_ERR_BAD_ARG, "positions or plan is NULL");
    return 0;
}

// Whether every vector of `v` elements that a kernel touches lies at a multiple of its size.
bool fits_vectors(const ps_heads_call* c, int v, bool backward)
{
    if (c->dim % v || (c->rotary / 2) % v) return false;
    const uintptr_t bytes = (uintptr_t)v * size_of(c->dtype);
    for (int w = 0; w < 2; ++w) {
        if (c->heads[w] == 0) continue;
        if ((uintptr_t)c->x[w] % bytes || (uintptr_t)c->out[w] % bytes) return false;
        for (int i = 0; i < 3; ++i)
            if (c->x_stride[w][i] % v) return false;
        if (!backward) continue;
        if ((uintptr_t)c->grad[w] % bytes) return false;
        for (int i = 0; i < 3; ++i)
            if (c->grad_stride[w][i] % v) return false;
    }
    return true;
}

struct HeadsShape {
    HeadsArgs a;
    int v;            // elements of a vector
    uint32_t blocks;  // of queries and keys together
    bool stream;      // the outputs are longer than the caches
};

// A wave's items of queries or keys, and the workgroups that take them.
void shape_part(const ps_heads_call* c, int which, const HeadsArgs& a, uint32_t most_blocks, HeadsPart& part)
{
    part.x = c->x[which];
    part.grad = c->grad[which];
    part.out = c->out[which];
    part.weight = c->weight[which];
    memcpy(part.x_stride, c->x_stride[which], sizeof(part.x_stride));
    memcpy(part.grad_stride, c->grad_stride[which], sizeof(part.grad_stride));
    part.heads = c->heads[which];
    if (part.heads == 0) return;
    part.weight_vectors = (uintptr_t)part.weight % 16 == 0;
    while ((1 << part.slot_shift) < part.heads && part.slot_shift < 6 - a.group_shift) ++part.slot_shift;
    const int tokens_shift = 6 - a.group_shift - part.slot_shift;
    const uint32_t waves = (uint32_t)(((uint64_t)a.all_tokens + (1u << tokens_shift) - 1) >> tokens_shift);
    // few tokens: a token's heads are spread over more waves, each of which makes the token's angles for itself
    while ((part.heads >> (part.slot_shift + part.split_shift)) > 1 && ((uint64_t)waves << part.split_shift) < 8 * kCus) ++part.split_shift;
    part.items = waves << part.split_shift;
    part.blocks = std::min((part.items + kHeadsWaves - 1) / kHeadsWaves, most_blocks);
}

HeadsShape heads_shape(const ps_heads_call* c, bool backward)
{
    HeadsShape s;
    HeadsArgs& a = s.a;
    memset(&a, 0, sizeof(a));
    memcpy(a.position_stride, c->position_stride, sizeof(a.position_stride));
    a.positions = c->positions;
    a.plan = c->plan;
    a.tokens = (uint32_t)c->tokens;
    a.all_tokens = (uint32_t)(c->batch * c->tokens);
    a.dim = c->dim;
    a.pairs = c->rotary / 2;
    a.eps = c->eps;
    a.inv_dim = 1.0f / (float)c->dim;
    a.weight_f32 = c->weight_dtype == PS_F32;
    a.positions_64 = c->position_bytes == 8;
    a.one_axis = c->axes == 1;
    a.interleaved = c->interleaved != 0;
    a.inverse = backward ? !c->inverse : c->inverse != 0;  // the gradient turns back
    // (8 bytes a lane of the 16-bit types: with 16, half as many waves fit a CU, and the norm's gradient took 131 us instead of 102)
    s.v = 4;
    while (!fits_vectors(c, s.v, backward)) s.v /= 2;
    a.whole = a.interleaved && fits_vectors(c, 2 * s.v, backward);
    const int units = (c->dim + 2 * s.v - 1) / (2 * s.v);
    while ((1 << a.group_shift) < units && a.group_shift < 6) ++a.group_shift;
    const uint32_t most = backward ? kBackwardBlocks : kForwardBlocks;
    const int heads = std::max(1, c->heads[0] + c->heads[1]);
    for (int which = 0; which < 2; ++which)
        shape_part(c, which, a, std::max(1u, (uint32_t)((uint64_t)most * c->heads[which] / heads)), a.part[which]);
    s.blocks = a.part[0].blocks + a.part[1].blocks;
    s.stream = c->batch * c->tokens * (c->heads[0] + c->heads[1]) * (int64_t)c->dim * size_of(c->dtype) > kCachedBytes;
    return s;
}

// Calls f(first, second) with both as constants.
template <typename F>
void with_flags(bool first, bool second, F f)
{
    if (first && second) return f(std::true_type(), std::true_type());
    if (first) return f(std::true_type(), std::false_type());
    if (second) return f(std::false_type(), std::true_type());
    f(std::false_type(), std::false_type());
}

// Calls f(type, vector length, units a lane).
template <typename F>
void with_heads_kernel(int dtype, int v, F f)
{
    with_type(dtype, [&](auto t) {
        if (v == 4) return f(t, Int<4>(), Int<1>());
        if (v == 2) return f(t, Int<2>(), Int<2>());
        f(t, Int<1>(), Int<4>());
    });
}
static_assert(PS_MAX_HEAD_DIM <= 2 * 4 * 64 && PS_MAX_HEAD_DIM <= 2 * 2 * 2 * 64 && PS_MAX_HEAD_DIM <= 2 * 1 * 4 * 64, "a group holds a head");

bool wants_weight_grad(const ps_heads_call* c)
{
    return (c->weight_grad[0] && c->heads[0]) || (c->weight_grad[1] && c->heads[1]);
}

// ------------------------------------------------------------------------------------------------------------- logits

// Calls f(vectors a thread keeps, threads), with at least `threads` of them: the shortest row that holds the vocabulary; 0 where
// none does.
template <typename T, typename F>
void with_row(int vocab, int threads, F f)
{
    const int vectors = vocab / (16 / (int)sizeof(T)) + 1;
    if (threads <= 256) {
        if (vectors <= 256) return f(Int<1>(), Int<256>());
        if (vectors <= 512) return f(Int<2>(), Int<256>());
        if (vectors <= 1024) return f(Int<4>(), Int<256>());
        if (vectors <= 2048) return f(Int<8>(), Int<256>());
    }
    if (threads <= 512) {
        if (vectors <= 4096) return f(Int<8>(), Int<512>());
        // (a few registers less are a workgroup more on a CU)
        if (vectors <= 6144) return f(Int<12>(), Int<512>());
        if (vectors <= 7168) return f(Int<14>(), Int<512>());
        if (vectors <= 8192) return f(Int<16>(), Int<512>());
    }
    if (vectors <= 4096) return f(Int<4>(), Int<1024>());
    if (vectors <= 16384) return f(Int<16>(), Int<1024>());
    f(Int<0>(), Int<1024>());
}

// Calls launch(first row, workgroups) for all rows: a workgroup each, and no more than a grid takes.
template <typename F>
int for_rows(int64_t rows, F launch)
{
    constexpr int64_t kMost = 1 << 21;
    for (int64_t first = 0; first < rows; first += kMost) {
        launch(first, dim3((unsigned)std::min(rows - first, kMost)));
        PS_HIP(hipGetLastError());
    }
    return 0;
}

constexpr int64_t kCountedRows = 1024;  // counted by every workgroup: 8 KiB of labels; more are counted by a kernel in front (2 us and a launch)
constexpr int64_t kMaxTopVocab = 1 << 30;
constexpr int64_t kMaxDistillVocab = 400000;  // a bit each in LDS, beside a list

int check_rows(int64_t rows, int64_t vocab, int64_t most, int dtype, const void* logits, int k)
{
    if (!known(dtype)) return fail(PS_ERR_BAD_ARG, "dtype %d is unknown", dtype);
    if (rows < 0) return fail(PS_ERR_BAD_ARG, "rows = %lld is negative", (long long)rows);
    if (vocab < 1 || vocab > most) return fail(PS_ERR_BAD_ARG, "vocab = %lld is not in 1 .. %lld", (long long)vocab, (long long)most);
    if (k < 1 || k > PS_MAX_TOP) return fail(PS_ERR_BAD_ARG, "k = %d is not in 1 .. %d", k, PS_MAX_TOP);
    if (rows && !logits) return fail(PS_ERR_BAD_ARG, "logits is NULL");
    if ((uintptr_t)logits % size_of(dtype)) return fail(PS_ERR_BAD_ARG, "logits is not aligned to its type");
    return 0;
}

// (and not beyond fp32, which the kernels use it in)
bool positive(double t) { return (float)t > 0.0f && std::isfinite((float)t) && std::isfinite((float)(1.4426950408889634 / t)); }

int distill_args(const ps_distill_call* c, bool backward, DistillArgs& a)
{
    if (!c) return fail(PS_ERR_BAD_ARG, "call is NULL");
    if (int rc = check_rows(c->rows, c->vocab, kMaxDistillVocab, c->dtype, c->logits, c->k)) return rc;
    if (!known(c->values_dtype)) return fail(PS_ERR_BAD_ARG, "values_dtype %d is unknown", c->values_dtype);
    if (c->ids_bytes != 4 && c->ids_bytes != 8) return fail(PS_ERR_BAD_ARG, "ids_bytes = %d", c->ids_bytes);
    if (c->labels && c->labels_bytes != 4 && c->labels_bytes != 8) return fail(PS_ERR_BAD_ARG, "labels_bytes = %d", c->labels_bytes);
    if (!positive(c->temperature)) return fail(PS_ERR_BAD_ARG, "temperature = %g must be positive", c->temperature);
    if (!(c->label_weight >= 0.0f && c->label_weight <= 1.0f))
        return fail(PS_ERR_BAD_ARG, "label_weight = %g is not in 0 .. 1", (double)c->label_weight);
    if (c->label_weight > 0.0f && !c->labels) return fail(PS_ERR_BAD_ARG, "label_weight without labels");
    if (c->rows && (!c->ids || !c->values)) return fail(PS_ERR_BAD_ARG, "the teacher's list is NULL");
    if (c->rows && !backward && !c->row_loss) return fail(PS_ERR_BAD_ARG, "row_loss is NULL");
    if (c->rows && backward && (!c->grad || !c->stats || !c->upstream)) return fail(PS_ERR_BAD_ARG, "grad, stats or upstream is NULL");
    if (c->mean && !c->denominator) return fail(PS_ERR_BAD_ARG, "a mean needs the denominator's place");
    memset(&a, 0, sizeof(a));
    a.logits = c->logits;
    a.ids = c->ids;
    a.values = c->values;
    a.teacher_lse = c->teacher_lse;
    a.labels = c->labels;
    a.row_loss = c->row_loss;
    a.stats = c->stats;
    // how many rows a mean is over: all of them, or as many as have a label, counted on the GPU
    a.denominator = c->mean && c->labels ? c->denominator : nullptr;
    a.count = c->mean ? (float)std::max<int64_t>(c->rows, 1) : 1.0f;
    a.count_rows = a.denominator && !backward && c->rows > 0 && c->rows <= kCountedRows;
    a.grad = c->grad;
    a.upstream = c->upstream;
    a.upstream_used = c->upstream_used;
    a.rows = c->rows;
    a.row_stride = c->row_stride;
    a.ids_stride = c->ids_stride;
    a.values_stride = c->values_stride;
    a.upstream_stride = c->upstream_stride;
    a.ignore_index = c->ignore_index;
    a.vocab = (int)c->vocab;
    a.k = c->k;
    a.values_dtype = c->values_dtype;
    a.factor = (float)(1.4426950408889634 / c->temperature);
    a.factor_low = (float)(1.4426950408889634 / c->temperature - (double)a.factor);
    a.temperature = c->temperature;
    a.inv_temperature = 1.0 / c->temperature;
    a.temperature_f = (float)c->temperature;
    a.label_weight = c->label_weight;
    a.upstream_value = c->upstream_value;
    a.ids_64 = c->ids_bytes == 8;
    a.labels_64 = c->labels_bytes == 8;
    return 0;
}

}  // namespace

extern "C" {

int ps_rotate_heads(const ps_heads_call* call, ps_stream_t stream)
{
    if (int rc = check_heads(call, false)) return rc;
    if (call->batch * call->tokens == 0 || call->heads[0] + call->heads[1] == 0) return 0;
    const HeadsShape s = heads_shape(call, false);
    with_heads_kernel(call->dtype, s.v, [&](auto t, auto v, auto u) {
        typedef decltype(t) T;
        const hipStream_t st = static_cast<hipStream_t>(stream);
        with_flags(call->norm, s.stream, [&](auto norm, auto streamed) {
            hipLaunchKernelGGL((rotate_heads_kernel<T, v(), u(), norm(), streamed()>), dim3(s.blocks), dim3(kHeadsBlock), 0, st, s.a);
        });
    });
    PS_HIP(hipGetLastError());
    return 0;
}

size_t ps_norm_rotate_heads_workspace_bytes(const ps_heads_call* call)
{
    if (check_heads(call, true) || call->batch * call->tokens == 0 || !wants_weight_grad(call)) return 0;
    return (size_t)heads_shape(call, true).blocks * (size_t)call->dim * sizeof(float);
}

int ps_norm_rotate_heads_backward(const ps_heads_call* call, void* d_workspace, size_t workspace_bytes, ps_stream_t stream)
{
    if (int rc = check_heads(call, true)) return rc;
    const size_t needed = ps_norm_rotate_heads_workspace_bytes(call);
    if (workspace_bytes < needed || (needed && (!d_workspace || (uintptr_t)d_workspace % 16)))
        return fail(PS_ERR_BAD_ARG, "the workspace has %zu bytes at %p, %zu are needed, 16-byte aligned", workspace_bytes, d_workspace, needed);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    WeightGrads sums;
    memset(&sums, 0, sizeof(sums));  // (of no tokens: zeros)
    if (call->batch * call->tokens > 0 && call->heads[0] + call->heads[1] > 0) {
        HeadsShape s = heads_shape(call, true);
        if (needed) {
            float* partial = static_cast<float*>(d_workspace);
            for (int which = 0; which < 2; ++which) {
                sums.partial[which] = s.a.part[which].partial = partial;
                sums.rows[which] = (int)s.a.part[which].blocks;
                partial += (size_t)s.a.part[which].blocks * (size_t)call->dim;
            }
        }
        with_heads_kernel(call->dtype, s.v, [&](auto t, auto v, auto u) {
            typedef decltype(t) T;
            with_flags(s.stream, false, [&](auto streamed, auto) {
                hipLaunchKernelGGL((norm_rotate_heads_backward_kernel<T, v(), u(), streamed()>), dim3(s.blocks), dim3(kHeadsBlock), 0, st, s.a);
            });
        });
        PS_HIP(hipGetLastError());
    }
    if (call->weight_grad[0] || call->weight_grad[1]) {
        sums.out[0] = call->weight_grad[0];
        sums.out[1] = call->weight_grad[1];
        sums.dim = call->dim;
        sums.f32 = call->weight_dtype == PS_F32;
        with_type(call->dtype, [&](auto t) {
            typedef decltype(t) T;
            hipLaunchKernelGGL((sum_weight_grads_kernel<T>), dim3((call->dim + kSumColumns - 1) / kSumColumns, 2), dim3(kSumColumns * kSumSlices),
                               0, st, sums);
        });
        PS_HIP(hipGetLastError());
    }
    return 0;
}

int ps_top_logits(const ps_top_call* call, ps_stream_t stream)
{
    if (!call) return fail(PS_ERR_BAD_ARG, "call is NULL");
    if (int rc = check_rows(call->rows, call->vocab, kMaxTopVocab, call->dtype, call->logits, call->k)) return rc;
    if (call->k > call->vocab) return fail(PS_ERR_BAD_ARG, "k = %d is more than the vocabulary of %lld", call->k, (long long)call->vocab);
    if (!positive(call->temperature)) return fail(PS_ERR_BAD_ARG, "temperature = %g must be positive", call->temperature);
    if (call->rows == 0) return 0;
    if (!call->values || !call->ids || !call->lse) return fail(PS_ERR_BAD_ARG, "values, ids or lse is NULL");
    TopArgs a;
    a.logits = call->logits;
    a.values = call->values;
    a.ids = call->ids;
    a.lse = call->lse;
    a.row_stride = call->row_stride;
    a.vocab = (int)call->vocab;
    a.k = call->k;
    a.factor = (float)(1.4426950408889634 / call->temperature);
    a.temperature = call->temperature;
    return for_rows(call->rows, [&](int64_t first, dim3 grid) {
        a.first_row = first;
        with_type(call->dtype, [&](auto t) {
            typedef decltype(t) T;
            with_row<T>(a.vocab, a.k <= 128 ? 256 : a.k <= 400 ? 512 : 1024, [&](auto nv, auto block) {
                hipLaunchKernelGGL((top_logits_kernel<T, nv(), block()>), grid, dim3(block()), 0, static_cast<hipStream_t>(stream), a);
            });
        });
    });
}

int ps_distill_loss(const ps_distill_call* call, ps_stream_t stream)
{
    DistillArgs a;
    if (int rc = distill_args(call, false, a)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a.denominator && !a.count_rows) {
        hipLaunchKernelGGL(count_rows_kernel, dim3(1), dim3(1024), 0, st, call->labels, a.labels_64, a.rows, a.ignore_index, call->denominator);
        PS_HIP(hipGetLastError());
    }
    const unsigned lds = 4u * (unsigned)member_words(a.vocab) + 12u * (unsigned)a.k;
    const int rc = for_rows(a.rows, [&](int64_t first, dim3 grid) {
        a.first_row = first;
        with_type(call->dtype, [&](auto t) {
            typedef decltype(t) T;
            with_row<T>(a.vocab, 256, [&](auto nv, auto block) {
                hipLaunchKernelGGL((distill_loss_kernel<T, nv(), block()>), grid, dim3(block()), lds, st, a);
            });
        });
    });
    if (rc) return rc;
    if (call->loss) {
        hipLaunchKernelGGL(sum_rows_kernel, dim3(1), dim3(1024), 0, st, call->row_loss, a.rows, a.denominator, a.count, call->loss);
        PS_HIP(hipGetLastError());
    }
    return 0;
}

int ps_distill_loss_backward(const ps_distill_call* call, ps_stream_t stream)
{
    DistillArgs a;
    if (int rc = distill_args(call, true, a)) return rc;
    if (a.rows == 0) return 0;
    // (where the gradient is there already, the workgroups are all it costs)
    const dim3 grid((unsigned)std::min<int64_t>(a.rows, 8 * kCus));
    with_type(call->dtype, [&](auto t) {
        typedef decltype(t) T;
        hipLaunchKernelGGL((distill_backward_kernel<T, 256>), grid, dim3(256), 8u * (unsigned)a.k, static_cast<hipStream_t>(stream), a);
    });
    PS_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
