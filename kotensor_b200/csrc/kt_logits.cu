// kt_logits.cu -- kt_logits_process: penalties, biases and grammar masks on logits,
// with the greedy choice in the same pass.
//
// A CTA owns kSlice consecutive token ids of one row.  It counts the row's tokens
// that fall in its slice in shared memory (integer counts: any order of the atomics
// gives the same; bit 31 marks a token seen anywhere, the low bits its occurrences in
// the answer) while its logits are on their way, then each logit is changed in
// registers and written once: bound by the two streams of logits, 8 bytes each.  Few
// ids are counted or have a bias: a bit for every four ids says where, so that the
// tables behind it are neither cleared nor read elsewhere, and one test finds a new
// largest value among four.  The row's largest logit is merged over its CTAs by a 64-bit
// maximum of {ordered value, ~index}: any order gives the same winner, the lowest index
// among equal values.
// 256 rows of 151936: 50 us (6.3 TB/s) with nothing on, 51 with a mask, 63 with penalties
// over 1025 tokens, 59 with 300 biases, 103 with all: then a CTA's three phases over
// the lists, not memory, are what its SM waits for.  (256 threads to a CTA, slices of 4096
// ids: 120 to 126 with all, 48 to 61 with nothing; the touched logits computed by a
// phase of their own, once each: 105 with all, 68 with penalties.)  One row 6.5 us.
#include "kt_kv8.h"

namespace kt {
namespace {

constexpr int kThreads = 512;
constexpr int kVecs = 4;
constexpr int kSlice = kThreads * kVecs * 4;
constexpr uint32_t kSeen = 0x80000000u;
constexpr uint32_t kNoBias = 0xffffffffu;
constexpr int kEarly = 2;   // tokens of a thread that are loaded ahead
constexpr int kList = 512;  // tokens, biases of a slice that are listed

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
__global__ void __launch_bounds__(kThreads, 3) logits_kernel(const __grid_constant__ kt_logits_args a) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    // tables of the slice, set where `touched` has the bit of their four ids: occurrences
    // of each id, and the list index of its first bias
    extern __shared__ __align__(16) uint32_t counts[];
    uint32_t* const first_bias = counts + (kPenal ? kSlice : 0);
    __shared__ uint32_t touched[kSlice / 128];
    __shared__ int repeated;  // an id of the slice has several biases
    __shared__ float penalty[3];  // repetition, frequency, presence
    __shared__ int listed, listed_biases;
    __shared__ uint32_t list[kPenal ? kList : 1];  // tokens of the slice, kSeen: of the answer
    __shared__ int bias_list[kBiased ? kList : 1], bias_index[kBiased ? kList : 1];
    __shared__ float early_value[kBiased ? kThreads : 1];
    __shared__ uint32_t part[kThreads / 32], part_id[kThreads / 32];
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
    // what else the row needs is asked for now, to arrive with the logits: the mask's words
    // of each four ids, lengths and penalties
    const uint32_t* allowed = a.allowed != nullptr ? a.allowed + row * a.allowed_stride : nullptr;
    uint32_t mask[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int at = begin + (i * kThreads + threadIdx.x) * 4, word = max(at, 0) >> 5;
        mask[i] = allowed != nullptr && at < a.vocab ? allowed[word] : 0;
    }
    // and the first tokens and biases of each thread, whatever the lists' lengths are
    const int32_t* tokens = a.tokens + row * a.token_stride;
    const int32_t* bias_ids = a.bias_ids + row * a.bias_stride;
    const float* bias_values = a.bias_values + row * a.bias_stride;
    int early[kEarly], early_id = -1;
    float early_bias = 0.0f;
    if (kPenal) {
#pragma unroll
        for (int i = 0; i < kEarly; ++i) {
            const int k = i * kThreads + static_cast<int>(threadIdx.x);
            early[i] = k < a.token_width ? tokens[k] : -1;
        }
    }
    if (kBiased && threadIdx.x < a.bias_width) {
        early_id = bias_ids[threadIdx.x];
        early_bias = bias_values[threadIdx.x];
    }
    const int biases = !kBiased ? 0 : a.bias_counts != nullptr ? min(a.bias_counts[row], a.bias_width) : a.bias_width;
    const int length = kPenal ? min(a.lengths[row], a.token_width) : 0;
    const int prompt = kPenal && a.prompt_lengths != nullptr ? a.prompt_lengths[row] : 0;
    if (kPenal || kBiased) {
        const int low = max(begin, 0), high = min(begin + kSlice, a.vocab);  // ids of this slice, and of the row
        auto each_token = [&](auto f) {
#pragma unroll
            for (int i = 0; i < kEarly; ++i) {
                const int k = i * kThreads + static_cast<int>(threadIdx.x);
                if (k < length && early[i] >= low && early[i] < high) f(k, early[i] - begin);
            }
#pragma unroll 4
            for (int k = kEarly * kThreads + threadIdx.x; k < length; k += kThreads) {
                const int id = tokens[k];
                if (id >= low && id < high) f(k, id - begin);
            }
        };
        auto each_bias = [&](auto f) {
            for (int k = threadIdx.x; k < biases; k += kThreads) {
                const int id = k < kThreads ? early_id : bias_ids[k];
                if (id >= low && id < high) f(k, id - begin);
            }
        };
        if (threadIdx.x < kSlice / 128) touched[threadIdx.x] = 0;
        if (threadIdx.x == 0) repeated = listed = listed_biases = 0;
        if (kPenal && threadIdx.x < 3) {
            const float* from = threadIdx.x == 0 ? a.repetition : threadIdx.x == 1 ? a.frequency : a.presence;
            penalty[threadIdx.x] = from != nullptr ? from[row] : threadIdx.x == 0 ? 1.0f : 0.0f;
        }
        __syncthreads();
        auto touch = [&](int at) {
            atomicOr(touched + at / 128, 1u << (at / 4 % 32));
            if (kPenal) *reinterpret_cast<uint4*>(counts + (at & ~3)) = make_uint4(0, 0, 0, 0);
            if (kBiased) *reinterpret_cast<uint4*>(first_bias + (at & ~3)) = make_uint4(kNoBias, kNoBias, kNoBias, kNoBias);
        };
        // what falls in the slice is listed, so that the lists are read from memory once
        if (kPenal)
            each_token([&](int k, int at) {
                touch(at);
                const int place = atomicAdd(&listed, 1);
                if (place < kList) list[place] = k >= prompt ? at | kSeen : at;
            });
        if (kBiased) {
            each_bias([&](int k, int at) {
                touch(at);
                const int place = atomicAdd(&listed_biases, 1);
                if (place < kList) {
                    bias_list[place] = at;
                    bias_index[place] = k;
                }
            });
            early_value[threadIdx.x] = early_bias;
        }
        __syncthreads();
        if (kPenal) {
            auto count = [&](int at, bool answer) {
                if (answer) atomicAdd(counts + at, 1u);
                atomicOr(counts + at, kSeen);
            };
            if (listed <= kList) {
                for (int i = threadIdx.x; i < listed; i += kThreads) count(list[i] & ~kSeen, list[i] & kSeen);
            } else {
                each_token([&](int k, int at) { count(at, k >= prompt); });
            }
        }
        if (kBiased) {
            auto claim = [&](int k, int at) {
                if (atomicMin(first_bias + at, static_cast<uint32_t>(k)) != kNoBias) repeated = 1;
            };
            if (listed_biases <= kList) {
                for (int i = threadIdx.x; i < listed_biases; i += kThreads) claim(bias_index[i], bias_list[i]);
            } else {
                each_bias(claim);
            }
        }
        __syncthreads();
    }

    float best = -1e9f;
    int best_id = 0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int local = (i * kThreads + threadIdx.x) * 4, at = begin + local;
        float w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        if ((kPenal || kBiased) && touched[local / 128] >> (local / 4 % 32) & 1) {
            if (kPenal) {
                const uint4 c = *reinterpret_cast<const uint4*>(counts + local);
                const uint32_t n[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (n[j] == 0) continue;
                    w[j] = w[j] > 0.0f ? __fdiv_rn(w[j], penalty[0]) : __fmul_rn(w[j], penalty[0]);
                    const uint32_t made = n[j] & ~kSeen;
                    if (made != 0) {
                        w[j] = __fsub_rn(w[j], __fmul_rn(penalty[1], static_cast<float>(made)));
                        w[j] = __fsub_rn(w[j], penalty[2]);
                    }
                }
            }
            if (kBiased) {
                const uint4 c = *reinterpret_cast<const uint4*>(first_bias + local);
                const uint32_t first[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (first[j] == kNoBias) continue;
                    w[j] = __fadd_rn(w[j], first[j] < kThreads ? early_value[first[j]] : bias_values[first[j]]);
                    if (repeated)  // the id's other entries, in list order
                        for (int k = static_cast<int>(first[j]) + 1; k < biases; ++k)
                            if (bias_ids[k] == at + j) w[j] = __fadd_rn(w[j], bias_values[k]);
                }
            }
        }
        if (allowed != nullptr) {
            uint32_t bits = at < 0 ? mask[i] << (-at & 31) : mask[i] >> (at & 31);
            if (at >= 0 && (at & 31) > 28 && at >> 5 < (a.vocab - 1) >> 5)  // four ids over two words: rows off the boundary only
                bits |= allowed[(at >> 5) + 1] << (32 - (at & 31));
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
    // the CTA's largest value, then the lowest of its ids
    auto reduce = [](uint32_t& value, uint32_t& id) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, value);
        id = __reduce_min_sync(0xffffffffu, value == top ? id : 0xffffffffu);
        value = top;
    };
    uint32_t value = best > -1e9f ? float_key(best) : 0, id = best_id;
    reduce(value, id);
    if (threadIdx.x % 32 == 0) {
        part[threadIdx.x / 32] = value;
        part_id[threadIdx.x / 32] = id;
    }
    __syncthreads();
    if (threadIdx.x >= 32) return;
    value = threadIdx.x < kThreads / 32 ? part[threadIdx.x] : 0;
    id = threadIdx.x < kThreads / 32 ? part_id[threadIdx.x] : 0xffffffffu;
    reduce(value, id);
    if (threadIdx.x != 0) return;
    const unsigned long long key = value == 0 ? 0 : static_cast<unsigned long long>(value) << 32 | (0xffffffffu - id);
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
        static std::atomic<uint64_t> allowed{0};
        const cudaError_t e = allow_shared(kernel, smem, allowed);
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
    const bool penalties = a.repetition || a.frequency || a.presence;
    if (((a.tokens || penalties) && !a.lengths) || (penalties && !a.tokens && a.token_width != 0))  // (a list of width 0 may have no address)
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
