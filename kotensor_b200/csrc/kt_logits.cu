// kt_logits.cu -- kt_logits_process: penalties, biases and grammar masks on logits,
// with the greedy choice in the same pass.
//
// A CTA owns kSlice consecutive token ids of one row.  It counts the row's tokens
// that fall in its slice in shared memory (integer counts: any order of the atomics
// gives the same; bit 31 marks a token seen anywhere, the low bits its occurrences in
// the answer) while its logits are on their way, then each logit is changed in
// registers and written once: bound by the two streams of logits, 8 bytes each.  What
// is rare, a counted token, a bias, a new largest value, is found by one test for four
// logits.  The row's largest logit is merged over its CTAs by a 64-bit maximum of
// {ordered value, ~index}: any order gives the same winner, the lowest index among
// equal values.
#include "kt_kv8.h"

namespace kt {
namespace {

constexpr int kThreads = 256;
constexpr int kVecs = 8;
constexpr int kSlice = kThreads * kVecs * 4;
constexpr uint32_t kSeen = 0x80000000u;
constexpr uint32_t kNoBias = 0xffffffffu;

// Larger floats give larger keys; -0 counts as 0.
__device__ __forceinline__ uint32_t float_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct RowScratch {
    unsigned long long best;
    uint32_t arrived, unused;
};

template <bool kPenal, bool kBiased>
__global__ void __launch_bounds__(kThreads) logits_kernel(const __grid_constant__ kt_logits_args a) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    // occurrences of each id of the slice, then the list index of its first bias
    extern __shared__ __align__(16) uint32_t counts[];
    uint32_t* const first_bias = counts + (kPenal ? kSlice : 0);
    __shared__ int repeated;  // an id of the slice has several biases
    __shared__ unsigned long long part[kThreads / 32];
    const int row = blockIdx.y;
    const float* x = a.logits + row * a.logits_stride;
    float* y = a.out + row * a.out_stride;
    // slices start on 16-byte boundaries of the row in memory
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(x) / 4 % 4);
    const bool same_skew = reinterpret_cast<uintptr_t>(y) / 4 % 4 == skew;
    const int begin = blockIdx.x * kSlice - skew;
    if (begin >= a.vocab) return;  // the skew of this row needs one slice fewer
    const bool whole = begin >= 0 && begin + kSlice <= a.vocab && same_skew;

    float4 v[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int at = begin + (i * kThreads + threadIdx.x) * 4;
        if (whole || (at >= 0 && at + 4 <= a.vocab)) {
            v[i] = *reinterpret_cast<const float4*>(x + at);
        } else {
            v[i].x = at >= 0 && at < a.vocab ? x[at] : -INFINITY;
            v[i].y = at + 1 >= 0 && at + 1 < a.vocab ? x[at + 1] : -INFINITY;
            v[i].z = at + 2 >= 0 && at + 2 < a.vocab ? x[at + 2] : -INFINITY;
            v[i].w = at + 3 >= 0 && at + 3 < a.vocab ? x[at + 3] : -INFINITY;
        }
    }
    if (kPenal || kBiased) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int at = (i * kThreads + threadIdx.x) * 4;
            if (kPenal) *reinterpret_cast<uint4*>(counts + at) = make_uint4(0, 0, 0, 0);
            if (kBiased) *reinterpret_cast<uint4*>(first_bias + at) = make_uint4(kNoBias, kNoBias, kNoBias, kNoBias);
        }
        if (threadIdx.x == 0) repeated = 0;
        __syncthreads();
    }
    // ids of this slice, and of the row
    const int low = max(begin, 0), high = min(begin + kSlice, a.vocab);
    if (kPenal) {
        const int32_t* tokens = a.tokens + row * a.token_stride;
        const int n = min(a.lengths[row], a.token_width), prompt = a.prompt_lengths != nullptr ? a.prompt_lengths[row] : 0;
#pragma unroll 8
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const int id = tokens[i];
            if (id < low || id >= high) continue;
            if (i >= prompt) atomicAdd(counts + id - begin, 1u);
            atomicOr(counts + id - begin, kSeen);
        }
    }
    const int32_t* bias_ids = a.bias_ids + row * a.bias_stride;
    const float* bias_values = a.bias_values + row * a.bias_stride;
    const int biases = !kBiased ? 0 : a.bias_counts != nullptr ? min(a.bias_counts[row], a.bias_width) : a.bias_width;
    if (kBiased) {
        for (int i = threadIdx.x; i < biases; i += kThreads) {
            const int id = bias_ids[i];
            if (id < low || id >= high) continue;
            if (atomicMin(first_bias + id - begin, static_cast<uint32_t>(i)) != kNoBias) repeated = 1;
        }
    }
    if (kPenal || kBiased) __syncthreads();

    const float repetition = kPenal && a.repetition != nullptr ? a.repetition[row] : 1.0f;
    const float frequency = kPenal && a.frequency != nullptr ? a.frequency[row] : 0.0f;
    const float presence = kPenal && a.presence != nullptr ? a.presence[row] : 0.0f;
    const uint32_t* allowed = a.allowed != nullptr ? a.allowed + row * a.allowed_stride : nullptr;
    float best = -1e9f;
    int best_id = 0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int local = (i * kThreads + threadIdx.x) * 4, at = begin + local;
        float w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        if (kPenal) {
            const uint4 c = *reinterpret_cast<const uint4*>(counts + local);
            if ((c.x | c.y | c.z | c.w) != 0) {
                const uint32_t n[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (n[j] == 0) continue;
                    w[j] = w[j] > 0.0f ? __fdiv_rn(w[j], repetition) : __fmul_rn(w[j], repetition);
                    const uint32_t made = n[j] & ~kSeen;
                    if (made != 0) {
                        w[j] = __fsub_rn(w[j], __fmul_rn(frequency, static_cast<float>(made)));
                        w[j] = __fsub_rn(w[j], presence);
                    }
                }
            }
        }
        if (kBiased) {
            const uint4 c = *reinterpret_cast<const uint4*>(first_bias + local);
            if ((c.x & c.y & c.z & c.w) != kNoBias) {
                const uint32_t first[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (first[j] == kNoBias) continue;
                    w[j] = __fadd_rn(w[j], bias_values[first[j]]);
                    if (repeated)  // the id's other entries, in list order
                        for (int k = static_cast<int>(first[j]) + 1; k < biases; ++k)
                            if (bias_ids[k] == at + j) w[j] = __fadd_rn(w[j], bias_values[k]);
                }
            }
        }
        if (allowed != nullptr && at + 3 >= 0 && at < a.vocab) {
            uint32_t bits;
            if (at >= 0) {
                const int word = at >> 5, last = (a.vocab - 1) >> 5;
                const uint32_t w0 = allowed[word];
                bits = w0 >> (at & 31);
                if ((at & 31) > 28 && word < last) bits = __funnelshift_r(w0, allowed[word + 1], at & 31);
            } else {
                bits = allowed[0] << -at;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (!(bits >> j & 1)) w[j] = -INFINITY;
        }
        const float top = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));  // of those that are not NaN
        if (top > best) {  // in the order of ids: the first of equal ones stays
            best = top;
            best_id = at + (w[0] == top ? 0 : w[1] == top ? 1 : w[2] == top ? 2 : 3);
        }
        if (whole || (same_skew && at >= 0 && at + 4 <= a.vocab)) {
            *reinterpret_cast<float4*>(y + at) = make_float4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at + j >= 0 && at + j < a.vocab) y[at + j] = w[j];
        }
    }
    if (a.next_token == nullptr) return;
    unsigned long long key = best > -1e9f ? static_cast<unsigned long long>(float_key(best)) << 32 | (0xffffffffu - best_id) : 0;
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
        key = key > other ? key : other;
    }
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = key;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < kThreads / 32; ++i) key = key > part[i] ? key : part[i];
    RowScratch* r = static_cast<RowScratch*>(a.scratch) + row;
    atomicMax(&r->best, key);
    const int slices = (a.vocab + skew + kSlice - 1) / kSlice;
    if (dev::atomic_add_acq_rel(reinterpret_cast<int32_t*>(&r->arrived), 1) != slices - 1) return;
    const unsigned long long won = atomicExch(&r->best, 0ull);  // the last CTA of the row leaves zeros
    r->arrived = 0;
    a.next_token[row] = won == 0 ? 0 : static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(won));
}

template <bool kPenal, bool kBiased>
cudaError_t launch_logits(const kt_logits_args& a, cudaStream_t s) {
    constexpr size_t smem = static_cast<size_t>(kSlice) * 4 * (kPenal + kBiased);
    const auto kernel = logits_kernel<kPenal, kBiased>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
    }
    return launch_dependent(kernel, dim3((a.vocab + 3 + kSlice - 1) / kSlice, a.rows), dim3(kThreads), smem, s, a);
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
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        const cudaError_t e = a.tokens ? a.bias_ids ? launch_logits<true, true>(a, s) : launch_logits<true, false>(a, s)
                              : a.bias_ids ? launch_logits<false, true>(a, s) : launch_logits<false, false>(a, s);
        return entry_launch(e, "logits launch");
    });
}
