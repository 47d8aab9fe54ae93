// kt_logits.cu -- kt_logits_process: penalties, biases and grammar masks on logits,
// with the greedy choice in the same pass.
//
// A CTA owns kSlice consecutive token ids of one row.  It counts the row's tokens
// that fall in its slice in shared memory (integer atomics: any order gives the
// same counts; bit 31 marks a token seen anywhere, the low bits its occurrences in
// the answer), then each logit is read, changed and written once.  The row's largest
// logit is merged over its CTAs by a 64-bit maximum of {ordered value, ~index}: any
// order gives the same winner, the lowest index among equal values.
#include "kt_kv8.h"

namespace kt {
namespace {

constexpr int kThreads = 512;
constexpr int kVecs = 4;
constexpr int kSlice = kThreads * kVecs * 4;
constexpr uint32_t kSeen = 0x80000000u;

// Larger floats give larger keys; NaN gives 0 (never chosen), -0 counts as 0.
__device__ __forceinline__ uint32_t float_key(float x) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct RowScratch {
    unsigned long long best;
    uint32_t arrived, unused;
};

__global__ void __launch_bounds__(kThreads) logits_kernel(kt_logits_args a) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    extern __shared__ uint32_t counts[];  // [kSlice], then the slice's biases where the call has any
    float* bias = reinterpret_cast<float*>(counts + kSlice);
    const int row = blockIdx.y;
    const float* x = a.logits + row * a.logits_stride;
    float* y = a.out + row * a.out_stride;
    // slices start on 16-byte boundaries of the row in memory
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(x) / 4 % 4);
    const bool same_skew = reinterpret_cast<uintptr_t>(y) / 4 % 4 == skew;
    const int begin = blockIdx.x * kSlice - skew;
    const bool penal = a.tokens != nullptr, biased = a.bias_ids != nullptr;
    if (begin >= a.vocab) return;  // the skew of this row needs one slice fewer

    float4 v[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int at = begin + (i * kThreads + threadIdx.x) * 4;
        if (at >= 0 && at + 4 <= a.vocab) {
            v[i] = *reinterpret_cast<const float4*>(x + at);
        } else {
            v[i].x = at >= 0 && at < a.vocab ? x[at] : 0.0f;
            v[i].y = at + 1 >= 0 && at + 1 < a.vocab ? x[at + 1] : 0.0f;
            v[i].z = at + 2 >= 0 && at + 2 < a.vocab ? x[at + 2] : 0.0f;
            v[i].w = at + 3 >= 0 && at + 3 < a.vocab ? x[at + 3] : 0.0f;
        }
    }
    if (penal || biased) {
        for (int i = threadIdx.x; i < kSlice; i += kThreads) {
            counts[i] = 0;
            if (biased) bias[i] = 0.0f;
        }
        __syncthreads();
    }
    if (penal) {
        const int32_t* tokens = a.tokens + row * a.token_stride;
        const int n = min(a.lengths[row], a.token_width), prompt = a.prompt_lengths != nullptr ? a.prompt_lengths[row] : 0;
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const int id = tokens[i], at = id - begin;
            if (id < 0 || id >= a.vocab || at < 0 || at >= kSlice) continue;
            atomicOr(counts + at, kSeen);
            if (i >= prompt) atomicAdd(counts + at, 1u);
        }
    }
    if (biased) {
        // the first entry of an id adds up all its entries, in list order
        const int32_t* ids = a.bias_ids + row * a.bias_stride;
        const float* values = a.bias_values + row * a.bias_stride;
        const int n = a.bias_counts != nullptr ? min(a.bias_counts[row], a.bias_width) : a.bias_width;
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const int id = ids[i], at = id - begin;
            if (id < 0 || id >= a.vocab || at < 0 || at >= kSlice) continue;
            bool first = true;
            for (int j = 0; j < i && first; ++j) first = ids[j] != id;
            if (!first) continue;
            float sum = values[i];
            for (int j = i + 1; j < n; ++j)
                if (ids[j] == id) sum = __fadd_rn(sum, values[j]);
            bias[at] = sum;
        }
    }
    __syncthreads();

    const float repetition = penal && a.repetition != nullptr ? a.repetition[row] : 1.0f;
    const float frequency = penal && a.frequency != nullptr ? a.frequency[row] : 0.0f;
    const float presence = penal && a.presence != nullptr ? a.presence[row] : 0.0f;
    const uint32_t* allowed = a.allowed != nullptr ? a.allowed + row * a.allowed_stride : nullptr;
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int local = (i * kThreads + threadIdx.x) * 4, at = begin + local;
        float w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int id = at + j;
            if (id < 0 || id >= a.vocab) continue;
            if (penal) {
                const uint32_t n = counts[local + j];
                if (n != 0) {
                    w[j] = w[j] > 0.0f ? __fdiv_rn(w[j], repetition) : __fmul_rn(w[j], repetition);
                    const uint32_t made = n & ~kSeen;
                    if (made != 0) {
                        w[j] = __fsub_rn(w[j], __fmul_rn(frequency, static_cast<float>(made)));
                        w[j] = __fsub_rn(w[j], presence);
                    }
                }
            }
            if (biased) w[j] = __fadd_rn(w[j], bias[local + j]);
            if (allowed != nullptr && !(allowed[id >> 5] >> (id & 31) & 1)) w[j] = -INFINITY;
            if (w[j] > -1e9f) {
                const unsigned long long key =
                    static_cast<unsigned long long>(float_key(w[j])) << 32 | (0xffffffffu - id);
                best = best > key ? best : key;
            }
        }
        if (same_skew && at >= 0 && at + 4 <= a.vocab) {
            *reinterpret_cast<float4*>(y + at) = make_float4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j >= 0 && at + j < a.vocab) y[at + j] = w[j];
        }
    }
    if (a.next_token == nullptr) return;
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = best > other ? best : other;
    }
    __shared__ unsigned long long part[kThreads / 32];
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = best;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < kThreads / 32; ++i) best = best > part[i] ? best : part[i];
    RowScratch* r = static_cast<RowScratch*>(a.scratch) + row;
    atomicMax(&r->best, best);
    const int slices = (a.vocab + skew + kSlice - 1) / kSlice;
    if (dev::atomic_add_acq_rel(reinterpret_cast<int32_t*>(&r->arrived), 1) != slices - 1) return;
    const unsigned long long won = atomicExch(&r->best, 0ull);  // the last CTA of the row leaves zeros
    r->arrived = 0;
    a.next_token[row] = won == 0 ? 0 : static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(won));
}

}  // namespace
}  // namespace kt

using namespace kt;

kt_status kt_logits_process(kt_ctx* ctx, const kt_logits_args* args, void* stream) {
    if (!ctx || !args) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    const kt_logits_args& a = *args;
    if (a.rows < 0 || a.rows > 65535) return entry_fail(KT_ERR_INVALID_ARGUMENT, "rows must be in 0..65535");
    if (a.vocab < 1 || a.vocab > 1 << 30) return entry_fail(KT_ERR_INVALID_ARGUMENT, "vocab must be in 1..2^30");
    if (a.rows == 0) return KT_OK;
    if (!a.logits || !a.out) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (a.logits_stride < a.vocab || a.out_stride < a.vocab)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "rows of the logits are shorter than vocab");
    if (a.tokens ? !a.lengths : (a.repetition || a.frequency || a.presence))
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "penalties need tokens and their lengths");
    if (!a.bias_ids != !a.bias_values)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "bias ids and values come together");
    if (a.token_stride < 0 || a.bias_stride < 0 || a.allowed_stride < 0 || a.token_width < 0 || a.bias_width < 0)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "strides and widths must not be negative");
    if (a.allowed && a.allowed_stride != 0 && a.allowed_stride < (a.vocab + 31) / 32)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "rows of the mask are shorter than vocab / 32 words");
    if (a.next_token && (!a.scratch || reinterpret_cast<uintptr_t>(a.scratch) % 16 != 0))
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "next_token needs 16-byte aligned scratch");
    if (a.rows > 1 && a.out == a.logits && a.out_stride != a.logits_stride)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "logits processed in place keep their stride");
    return c_entry(ctx, [&] {
        const size_t smem = static_cast<size_t>(kSlice) * 4 * (a.bias_ids ? 2 : 1);
        cudaError_t e = cudaSuccess;
        if (a.bias_ids)
            e = cudaFuncSetAttribute(logits_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSlice * 8);
        if (e == cudaSuccess)
            e = launch_dependent(logits_kernel, dim3((a.vocab + 3 + kSlice - 1) / kSlice, a.rows), dim3(kThreads), smem,
                                 static_cast<cudaStream_t>(stream), a);
        return entry_launch(e, "logits launch");
    });
}
