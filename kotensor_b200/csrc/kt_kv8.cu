// kt_kv8.cu -- the 8-bit key/value cache: storing tokens, advancing lengths and
// evicting tokens by accumulated attention weight, with their C entries (the
// attention is kt_kv8_attention.cu).
//
// One block of `block` slots of one head holds x as code * scale,
//   a = max |x|,  scale = a * (1/127),  code = rint(x * (127 * (1/a))),
// every step an fp32 operation rounded to nearest even, so that the result is one
// defined set of bits.  The magnitudes are compared as the bits of |x|: NaN orders
// above infinity there, so one comparison at the end finds a value that is not
// finite anywhere in the block.
#include "kt_kv8.h"

namespace kt {
namespace {

constexpr int kThreads = 256;
constexpr int kVecs = 64 * kKv8MaxHeadDim / 4 / kThreads;  // four-value pieces of a block a thread holds
constexpr uint32_t kTiny = 0x0d800000u;                     // bits of 2^-100
constexpr uint32_t kInf = 0x7f800000u;

struct BlockScale {
    float scale, inverse;  // inverse 0: all codes 0
};
__device__ __forceinline__ BlockScale block_scale(uint32_t top) {
    if (top >= kInf) return {__uint_as_float(0x7fc00000u), 0.0f};
    if (top < kTiny) return {0.0f, 0.0f};
    const float a = __uint_as_float(top);
    return {__fmul_rn(a, 1.0f / 127.0f), __fmul_rn(__frcp_rn(a), 127.0f)};
}
__device__ __forceinline__ int8_t code_of(float x, float inverse) {
    if (inverse == 0.0f) return 0;  // NaN and infinity times 0 are not 0
    return static_cast<int8_t>(fminf(fmaxf(rintf(__fmul_rn(x, inverse)), -127.0f), 127.0f));
}
__device__ __forceinline__ char4 codes_of(float4 x, float inverse) {
    return make_char4(code_of(x.x, inverse), code_of(x.y, inverse), code_of(x.z, inverse), code_of(x.w, inverse));
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t magnitude(float4 x) {
    return max(max(magnitude(x.x), magnitude(x.y)), max(magnitude(x.z), magnitude(x.w)));
}
// The largest value of the block's threads, in every thread; also a barrier.
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
    __shared__ uint32_t part[kThreads / 32];
    v = __reduce_max_sync(0xffffffffu, v);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    v = part[threadIdx.x % (kThreads / 32)];
    return __reduce_max_sync(0xffffffffu, v);
}
// Four floats at p, by one load where the address allows it.
__device__ __forceinline__ float4 load4(const float* p, bool aligned) {
    if (aligned) return *reinterpret_cast<const float4*>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}

// One CTA per (block that the new tokens touch, head, sequence, key or value).
// The block's values stay in registers between the search for the largest and
// their rounding: each is read once.  The CTA of a sequence's first touched block
// is the only one that reads the old tail and writes the new one.
__global__ void __launch_bounds__(kThreads) kv8_store_kernel(Kv8 c, const float* __restrict__ k,
                                                             const float* __restrict__ v, int64_t k_stride,
                                                             int64_t v_stride, int aligned, int rows_per_seq,
                                                             const int32_t* __restrict__ counts,
                                                             int32_t* __restrict__ status) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const int b = blockIdx.z >> 1, h = blockIdx.y, x = blockIdx.x;
    const bool value = blockIdx.z & 1;
    const int held = kv8_held(c, b);
    int n = kv8_rows(counts, b, rows_per_seq);
    if (n > c.capacity - held) {
        n = c.capacity - held;
        if (status != nullptr && threadIdx.x == 0 && x == 0 && h == 0 && !value) atomicOr(status, KT_ERR_INVALID_ARGUMENT);
    }
    if (n == 0) return;
    const int inside = held % c.block, first = held / c.block;
    if (x * c.block >= inside + n) return;
    const int d4 = c.head_dim / 4;
    const int64_t head = static_cast<int64_t>(b) * c.kv_heads + h;
    int8_t* codes = (value ? c.v_codes : c.k_codes) + (head * c.capacity + (first + x) * c.block) * c.head_dim;
    float* tail = (value ? c.v_tail : c.k_tail) + head * c.block * c.head_dim;
    const int64_t stride = value ? v_stride : k_stride;
    const float* rows = (value ? v : k) + static_cast<int64_t>(b) * rows_per_seq * stride + h * c.head_dim;

    float4 r[kVecs];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int e = i * kThreads + threadIdx.x, slot = e / d4, col = (e - slot * d4) * 4;
        const int row = x * c.block + slot - inside;  // negative: a slot that was held before (x == 0)
        r[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (slot < c.block && row < n)
            r[i] = row < 0 ? *reinterpret_cast<const float4*>(tail + slot * c.head_dim + col)
                           : load4(rows + row * stride + col, aligned);
        top = max(top, magnitude(r[i]));
    }
    const BlockScale s = block_scale(block_max(top));
    if (threadIdx.x == 0) (value ? c.v_scales : c.k_scales)[head * (c.capacity / c.block) + first + x] = s.scale;
    const int last = (held + n) / c.block;  // the new open block
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int e = i * kThreads + threadIdx.x, slot = e / d4, col = (e - slot * d4) * 4;
        const int row = x * c.block + slot - inside;
        if (slot >= c.block || row >= n) continue;
        *reinterpret_cast<char4*>(codes + slot * c.head_dim + col) = codes_of(r[i], s.inverse);
        if (x == 0 && last == first && row >= 0) *reinterpret_cast<float4*>(tail + slot * c.head_dim + col) = r[i];
    }
    if (x == 0 && last != first) {  // the rows left over after the last full block
        const int left = (held + n) % c.block;
        for (int e = threadIdx.x; e < left * d4; e += kThreads) {
            const int slot = e / d4, col = (e - slot * d4) * 4;
            *reinterpret_cast<float4*>(tail + slot * c.head_dim + col) =
                load4(rows + (n - left + slot) * stride + col, aligned);
        }
    }
    if (c.weights != nullptr && !value)
        for (int slot = threadIdx.x; slot < c.block; slot += kThreads) {
            const int row = x * c.block + slot - inside;
            if (row >= 0 && row < n) c.weights[head * c.capacity + held + row] = 0.0f;
        }
}

__global__ void kv8_advance_kernel(int32_t* __restrict__ lengths, int batch, int rows,
                                   const int32_t* __restrict__ counts, int limit) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    for (int b = threadIdx.x; b < batch; b += blockDim.x)
        lengths[b] = min(lengths[b] + (counts == nullptr ? rows : counts[b]), limit);
}

// ------------------------------------------------------------ eviction

constexpr int kSelectThreads = 1024;

// Weights ordered as unsigned integers: negative ones reversed below the others,
// -0 as 0, NaN above all.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Sum of v over the block; also a barrier on both sides.
__device__ __forceinline__ int block_sum(int v) {
    __shared__ int part[kSelectThreads / 32];
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, part[threadIdx.x % 32]);
}

// One CTA per (head, sequence): the smallest key of the kept candidates, found bit
// by bit from the top, then the kept slots in order into `order` and their weights
// to the front.
__global__ void __launch_bounds__(kSelectThreads) kv8_select_kernel(Kv8 c, int keep, int recent,
                                                                    int32_t* __restrict__ order) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const int b = blockIdx.y, h = blockIdx.x, held = kv8_held(c, b);
    if (held <= keep) return;
    const int64_t head = static_cast<int64_t>(b) * c.kv_heads + h;
    float* w = c.weights + head * c.capacity;
    order += head * c.capacity;
    const int candidates = held - recent, want = keep - recent;
    uint32_t bound = 0;  // the largest key that at least `want` candidates reach
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t trial = bound | (1u << bit);
        int n = 0;
        for (int i = threadIdx.x; i < candidates; i += kSelectThreads) n += order_key(w[i]) >= trial;
        if (block_sum(n) >= want) bound = trial;
    }
    int above = 0;
    for (int i = threadIdx.x; i < candidates; i += kSelectThreads) above += order_key(w[i]) > bound;
    const int ties = want - block_sum(above);  // how many of those equal to the bound are kept, lowest slots first
    __shared__ int kept_of[32], tied_of[32];
    int kept_before = 0, tied_before = 0;
    for (int base = 0; base < held; base += kSelectThreads) {
        const int i = base + threadIdx.x;
        const float x = i < held ? w[i] : 0.0f;
        const bool late = i >= candidates && i < held;
        const uint32_t key = i < candidates ? order_key(x) : 0;
        const bool tied = i < candidates && key == bound;
        const uint32_t tied_lanes = __ballot_sync(0xffffffffu, tied);
        const uint32_t before = (1u << (threadIdx.x % 32)) - 1;
        if (threadIdx.x % 32 == 0) tied_of[threadIdx.x / 32] = __popc(tied_lanes);
        __syncthreads();
        int rank = tied_before + __popc(tied_lanes & before), all_tied = 0;
        for (int o = 0; o < 32; ++o) {
            if (o < threadIdx.x / 32) rank += tied_of[o];
            all_tied += tied_of[o];
        }
        const bool keep_it = late || (i < candidates && (key > bound || (tied && rank < ties)));
        const uint32_t kept_lanes = __ballot_sync(0xffffffffu, keep_it);
        if (threadIdx.x % 32 == 0) kept_of[threadIdx.x / 32] = __popc(kept_lanes);
        __syncthreads();
        int place = kept_before + __popc(kept_lanes & before), all_kept = 0;
        for (int o = 0; o < 32; ++o) {
            if (o < threadIdx.x / 32) place += kept_of[o];
            all_kept += kept_of[o];
        }
        if (keep_it) {  // place <= i, and every weight up to this chunk's end has been read
            order[place] = i;
            w[place] = x;
        }
        kept_before += all_kept;
        tied_before += all_tied;
        __syncthreads();
    }
}

// One CTA per (head, sequence, key or value) walks the new blocks in order: the
// token that moves to slot i comes from a slot >= i, so what a block overwrites no
// later block still needs, and its own values are all in registers at the barrier.
__global__ void __launch_bounds__(kThreads) kv8_move_kernel(Kv8 c, int keep, const int32_t* __restrict__ order) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const int b = blockIdx.z >> 1, h = blockIdx.y;
    const bool value = blockIdx.z & 1;
    if (kv8_held(c, b) <= keep) return;
    const int64_t head = static_cast<int64_t>(b) * c.kv_heads + h;
    order += head * c.capacity;
    int8_t* codes = (value ? c.v_codes : c.k_codes) + head * c.capacity * c.head_dim;
    float* scales = (value ? c.v_scales : c.k_scales) + head * (c.capacity / c.block);
    float* tail = (value ? c.v_tail : c.k_tail) + head * c.block * c.head_dim;
    const int d4 = c.head_dim / 4;
    for (int base = 0; base < keep; base += c.block) {
        float4 r[kVecs];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int e = i * kThreads + threadIdx.x, slot = e / d4, col = (e - slot * d4) * 4;
            r[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (slot < c.block && base + slot < keep) {
                const int from = order[base + slot];
                const char4 q = *reinterpret_cast<const char4*>(codes + static_cast<int64_t>(from) * c.head_dim + col);
                const float s = scales[from / c.block];
                r[i] = make_float4(__fmul_rn(s, q.x), __fmul_rn(s, q.y), __fmul_rn(s, q.z), __fmul_rn(s, q.w));
            }
            top = max(top, magnitude(r[i]));
        }
        const BlockScale s = block_scale(block_max(top));
        if (threadIdx.x == 0) scales[base / c.block] = s.scale;
        const bool open = keep - base < c.block;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int e = i * kThreads + threadIdx.x, slot = e / d4, col = (e - slot * d4) * 4;
            if (slot >= c.block || base + slot >= keep) continue;
            *reinterpret_cast<char4*>(codes + static_cast<int64_t>(base + slot) * c.head_dim + col) =
                codes_of(r[i], s.inverse);
            if (open) *reinterpret_cast<float4*>(tail + slot * c.head_dim + col) = r[i];
        }
        __syncthreads();  // block_max's shared words are free again
    }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

const char* kv8_check(const Kv8* c) {
    if (c == nullptr || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales || !c->k_tail || !c->v_tail ||
        !c->lengths)
        return "NULL argument";
    if (c->batch < 1 || c->batch > 32767) return "batch must be in 1..32767";
    if (c->kv_heads < 1 || c->kv_heads > 65535) return "kv_heads must be in 1..65535";
    if (c->head_dim < 16 || c->head_dim > kKv8MaxHeadDim || c->head_dim % 16 != 0)
        return "head_dim must be a multiple of 16 in 16..128";
    if (c->block != 16 && c->block != 32 && c->block != 64) return "block must be 16, 32 or 64";
    if (c->capacity < c->block || c->capacity % c->block != 0) return "capacity must be a positive multiple of block";
    if (!aligned16(c->k_codes) || !aligned16(c->v_codes) || !aligned16(c->k_scales) || !aligned16(c->v_scales) ||
        !aligned16(c->k_tail) || !aligned16(c->v_tail) || !aligned16(c->weights))
        return "cache buffers must be 16-byte aligned";
    return nullptr;
}

}  // namespace kt

using namespace kt;

kt_status kt_kv8_store(kt_ctx* ctx, const kt_kv8_cache* cache, const float* k, const float* v, int64_t k_stride,
                       int64_t v_stride, int32_t rows_per_seq, const int32_t* counts, int32_t* status, void* stream) {
    if (!ctx) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (const char* why = kv8_check(cache)) return entry_fail(KT_ERR_INVALID_ARGUMENT, why);
    if (rows_per_seq < 0) return entry_fail(KT_ERR_INVALID_ARGUMENT, "Negative row count");
    if (rows_per_seq == 0) return KT_OK;
    if (!k || !v) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    const int64_t width = static_cast<int64_t>(cache->kv_heads) * cache->head_dim;
    if (k_stride < width || v_stride < width)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "rows of k and v are shorter than kv_heads * head_dim");
    return c_entry(ctx, [&] {
        const int aligned = aligned16(k) && aligned16(v) && k_stride % 4 == 0 && v_stride % 4 == 0;
        const int rows = std::min(rows_per_seq, cache->capacity);  // more would be dropped
        const dim3 grid((rows + cache->block - 1) / cache->block + 1, cache->kv_heads, 2 * cache->batch);
        return entry_launch(launch_dependent(kv8_store_kernel, grid, dim3(kThreads), 0,
                                             static_cast<cudaStream_t>(stream), *cache, k, v, k_stride, v_stride,
                                             aligned, rows_per_seq, counts, status),
                            "kv8 store launch");
    });
}

size_t kt_kv8_scratch_bytes(int32_t batch, int32_t rows_per_seq, int32_t heads, int32_t kv_heads, int32_t head_dim,
                            int32_t capacity, int32_t weights) {
    if (batch <= 0 || rows_per_seq <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || capacity <= 0) return 0;
    const size_t order = weights ? static_cast<size_t>(batch) * kv_heads * capacity * sizeof(int32_t) : 0;
    return kKv8CounterBytes +
           std::max(order, kv8_attention_bytes(batch, rows_per_seq, heads, kv_heads, head_dim, capacity, weights != 0));
}

kt_status kt_kv8_attention(kt_ctx* ctx, const kt_kv8_cache* cache, const float* q, int64_t q_stride, float* context,
                           int32_t rows_per_seq, const int32_t* counts, int32_t heads, float scale,
                           int32_t accumulate_weights, void* scratch, void* stream) {
    if (!ctx) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (const char* why = kv8_check(cache)) return entry_fail(KT_ERR_INVALID_ARGUMENT, why);
    if (rows_per_seq < 0) return entry_fail(KT_ERR_INVALID_ARGUMENT, "Negative row count");
    if (rows_per_seq == 0) return KT_OK;
    if (!q || !context || !scratch) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (heads < 1 || heads % cache->kv_heads != 0)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "heads must be a positive multiple of kv_heads");
    if (q_stride < static_cast<int64_t>(heads) * cache->head_dim)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "rows of q are shorter than heads * head_dim");
    if (accumulate_weights && !cache->weights)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "the cache keeps no weights to accumulate");
    if (!aligned16(scratch)) return entry_fail(KT_ERR_INVALID_ARGUMENT, "scratch must be 16-byte aligned");
    return c_entry(ctx, [&] {
        const Kv8Attention a{*cache, q, q_stride, context, counts, rows_per_seq, heads, scale, accumulate_weights, scratch};
        return entry_launch(launch_kv8_attention(a, ctx->sm_count, ctx->d_error, static_cast<cudaStream_t>(stream)),
                            "kv8 attention launch");
    });
}

kt_status kt_kv8_advance(kt_ctx* ctx, int32_t* lengths, int32_t batch, int32_t rows, const int32_t* counts,
                         int32_t limit, void* stream) {
    if (!ctx || !lengths) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (batch < 1 || limit < 0) return entry_fail(KT_ERR_INVALID_ARGUMENT, "bad advance arguments");
    return c_entry(ctx, [&] {
        return entry_launch(launch_dependent(kv8_advance_kernel, dim3(1), dim3(256), 0,
                                             static_cast<cudaStream_t>(stream), lengths, batch, rows, counts, limit),
                            "kv8 advance launch");
    });
}

kt_status kt_kv8_evict(kt_ctx* ctx, const kt_kv8_cache* cache, int32_t keep, int32_t recent, void* scratch,
                       void* stream) {
    if (!ctx) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (const char* why = kv8_check(cache)) return entry_fail(KT_ERR_INVALID_ARGUMENT, why);
    if (!scratch) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (!cache->weights) return entry_fail(KT_ERR_INVALID_ARGUMENT, "the cache keeps no weights to evict by");
    if (keep < 1 || recent < 0 || recent > keep)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "eviction needs 0 <= recent <= keep and 1 <= keep");
    if (!aligned16(scratch)) return entry_fail(KT_ERR_INVALID_ARGUMENT, "scratch must be 16-byte aligned");
    if (keep >= cache->capacity) return KT_OK;  // nothing can hold more
    return c_entry(ctx, [&] {
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        int32_t* order = reinterpret_cast<int32_t*>(static_cast<char*>(scratch) + kKv8CounterBytes);
        const dim3 heads(cache->kv_heads, cache->batch);
        cudaError_t e = launch_dependent(kv8_select_kernel, heads, dim3(kSelectThreads), 0, s, *cache, keep, recent,
                                         order);
        if (e == cudaSuccess)
            e = launch_dependent(kv8_move_kernel, dim3(1, cache->kv_heads, 2 * cache->batch), dim3(kThreads), 0, s,
                                 *cache, keep, order);
        return entry_launch(e, "kv8 evict launch");
    });
}
