// kt_kv8.h -- the 8-bit key/value cache as its kernels see it, and the
// launchers of kt_kv8.cu and kt_kv8_attention.cu.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <exception>
#include <new>
#include <string>

#include "kt_device.cuh"
#include "kt_internal.h"

namespace kt {

using Kv8 = kt_kv8_cache;  // passed to kernels by value

constexpr int kKv8MaxHeadDim = 128;

// Scratch layout (kt_kv8_scratch_bytes): the attention's merge counters at the
// front, at the same place for every call, then what one call uses freely.
constexpr size_t kKv8CounterBytes = 4096;  // (include/kt_cuda.h and kv8.py give this number)
constexpr int kKv8MaxCtas = static_cast<int>(kKv8CounterBytes / sizeof(int32_t));

// Runs a C entry's body: no C++ exception crosses the boundary, and the
// context's device is current inside (the caller's is put back).
template <typename Body>
kt_status c_entry(kt_ctx* ctx, Body body) {
    struct Restore {  // also where the body throws
        int device = -1;
        ~Restore() {
            if (device >= 0) cudaSetDevice(device);
        }
    };
    try {
        int before = 0;
        Restore restore;
        cudaError_t e = cudaGetDevice(&before);
        if (e == cudaSuccess && before != ctx->device) {
            restore.device = before;
            e = cudaSetDevice(ctx->device);
        }
        if (e != cudaSuccess) {
            set_error(std::string("cudaSetDevice: ") + cudaGetErrorString(e));
            return KT_ERR_CUDA;
        }
        return body();
    } catch (const std::bad_alloc&) {
        return KT_ERR_OUT_OF_MEMORY;
    } catch (...) {
        return KT_ERR_CUDA;
    }
}

inline kt_status entry_fail(kt_status st, const char* msg) {
    try {
        set_error(msg);
    } catch (...) {  // the status stands without its message
    }
    return st;
}

inline kt_status entry_launch(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return KT_OK;
    set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return e == cudaErrorMemoryAllocation ? KT_ERR_OUT_OF_MEMORY : KT_ERR_CUDA;
}

// A launch that may start while the previous kernel of its stream ends
// (programmatic dependent launch): every kernel launched by it waits
// (griddepcontrol.wait) before it touches memory.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                             Args... args) {
    cudaLaunchConfig_t lc = {};
    lc.gridDim = grid;
    lc.blockDim = block;
    lc.dynamicSmemBytes = smem;
    lc.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    return cudaLaunchKernelEx(&lc, kernel, static_cast<Params>(args)...);
}

// Lets `kernel` use `bytes` of dynamic shared memory; asked of the runtime once a
// device for each place of use (`done`, a static of the caller, has a bit for each).
template <typename Kernel>
cudaError_t allow_shared(Kernel kernel, size_t bytes, std::atomic<uint64_t>& done) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (device & 63);
    if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// NULL when the cache can be used, else what is wrong with it (kt_kv8.cu).
const char* kv8_check(const Kv8* c);

struct Kv8Attention {
    Kv8 cache;
    const float* q;
    int64_t q_stride;
    float* context;
    const int32_t* counts;
    int32_t rows_per_seq, heads;
    float scale;
    int32_t accumulate;
    void* scratch;
};
// Bytes behind the counters that the attention of these sizes uses (kt_kv8_attention.cu).
size_t kv8_attention_bytes(int32_t batch, int32_t rows_per_seq, int32_t heads, int32_t kv_heads, int32_t head_dim,
                           int32_t capacity, bool weights);
cudaError_t launch_kv8_attention(const Kv8Attention& a, int sm_count, int32_t* err, cudaStream_t s);
// Many query rows, on tcgen05 (kt_kv8_prompt.cu).  aligned: bit 0, q's rows lie on
// 16-byte boundaries.  lse (NULL: not wanted): ln of the softmax's sum of every row
// and head.  parts: kv8_prompt_bytes of scratch, used where a launch of fewer CTAs than
// SMs splits the slots into kv8_prompt_splits parts.
constexpr int kPromptCtas = 148;
int kv8_prompt_splits(int32_t batch, int32_t rows_per_seq, int32_t heads, int32_t kv_heads, int32_t capacity);
size_t kv8_prompt_bytes(int32_t head_dim);
cudaError_t launch_kv8_prompt(const Kv8Attention& a, int aligned, float* parts, float* lse, int32_t* err, cudaStream_t s);

#ifdef __CUDACC__
// Tokens that sequence b holds, whatever the caller left in lengths.
__device__ __forceinline__ int kv8_held(const Kv8& c, int b) {
    return min(max(c.lengths[b], 0), c.capacity);
}
// Rows of this call that sequence b adds or asks with.
__device__ __forceinline__ int kv8_rows(const int32_t* counts, int b, int rows_per_seq) {
    return counts == nullptr ? rows_per_seq : min(max(counts[b], 0), rows_per_seq);
}
#endif

}  // namespace kt
