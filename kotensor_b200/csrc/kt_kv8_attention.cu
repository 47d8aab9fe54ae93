// kt_kv8_attention.cu -- attention over the 8-bit key/value cache.
//
// Row t of sequence b with n = lengths[b]: for each query head, over slots
// j <= n + t,  s_j = scale * (q . K_j),  out = sum_j softmax(s)_j V_j, with
// K_j = code * scale of the slot's block.
#include "kt_kv8.h"

namespace kt {
namespace {

constexpr int kWarps = 8;
constexpr int kDims = kKv8MaxHeadDim / 32;  // dims a lane holds

// One CTA per (row, query head, sequence): warp w takes slots w, w + 8, ..., a lane
// dims lane, lane + 32, ...; each warp keeps a running maximum, sum and weighted
// sum of values, merged at the end.
__global__ void __launch_bounds__(kWarps * 32) kv8_attention_rows_kernel(Kv8Attention a, float* __restrict__ lse) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const Kv8& c = a.cache;
    const int t = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, d = c.head_dim;
    const int64_t row = static_cast<int64_t>(b) * a.rows_per_seq + t;
    float* out = a.context + (row * a.heads + head) * d;
    if (t >= kv8_rows(a.counts, b, a.rows_per_seq)) {
        for (int i = threadIdx.x; i < d; i += blockDim.x) out[i] = 0.0f;
        return;
    }
    const int n = min(kv8_held(c, b) + t + 1, c.capacity);
    const int64_t kvh = static_cast<int64_t>(b) * c.kv_heads + head / (a.heads / c.kv_heads);
    const int8_t* kc = c.k_codes + kvh * c.capacity * d;
    const int8_t* vc = c.v_codes + kvh * c.capacity * d;
    const float* ks = c.k_scales + kvh * (c.capacity / c.block);
    const float* vs = c.v_scales + kvh * (c.capacity / c.block);
    const float* q = a.q + row * a.q_stride + head * d;
    float qr[kDims], o[kDims] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kDims; ++i) qr[i] = lane + 32 * i < d ? q[lane + 32 * i] : 0.0f;
    for (int j = warp; j < n; j += kWarps) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kDims; ++i)
            if (lane + 32 * i < d) s = fmaf(qr[i], kc[static_cast<int64_t>(j) * d + lane + 32 * i], s);
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s = s * ks[j / c.block] * a.scale;
        const float top = fmaxf(m, s), keep = m == top ? 1.0f : expf(m - top), p = s == -INFINITY ? 0.0f : expf(s - top);
        const float pv = p * vs[j / c.block];
        l = l * keep + p;
        m = top;
#pragma unroll
        for (int i = 0; i < kDims; ++i)
            if (lane + 32 * i < d) o[i] = o[i] * keep + pv * vc[static_cast<int64_t>(j) * d + lane + 32 * i];
    }
    __shared__ float sm[kWarps], sl[kWarps], so[kWarps][kKv8MaxHeadDim];
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (int i = 0; i < kDims; ++i) so[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float top = -INFINITY, sum = 0.0f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w]);
    for (int w = 0; w < kWarps; ++w) sum += sl[w] > 0.0f || sl[w] != sl[w] ? sl[w] * expf(sm[w] - top) : 0.0f;
    for (int i = threadIdx.x; i < d; i += blockDim.x) {
        float y = 0.0f;
        for (int w = 0; w < kWarps; ++w)
            if (sl[w] > 0.0f || sl[w] != sl[w]) y += so[w][i] * expf(sm[w] - top);
        out[i] = y / sum;
    }
    if (threadIdx.x == 0) lse[row * a.heads + head] = top + logf(sum);
}

// One warp per slot adds up its weight over the rows and heads of its group, in order.
__global__ void __launch_bounds__(kWarps * 32) kv8_weights_kernel(Kv8Attention a, const float* __restrict__ lse) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const Kv8& c = a.cache;
    const int j = blockIdx.x * kWarps + threadIdx.x / 32, h = blockIdx.y, b = blockIdx.z;
    const int lane = threadIdx.x % 32, d = c.head_dim, group = a.heads / c.kv_heads;
    const int rows = kv8_rows(a.counts, b, a.rows_per_seq), held = kv8_held(c, b);
    if (j >= min(held + rows, c.capacity)) return;
    const int64_t kvh = static_cast<int64_t>(b) * c.kv_heads + h;
    float k[kDims], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kDims; ++i)
        k[i] = lane + 32 * i < d ? c.k_codes[(kvh * c.capacity + j) * d + lane + 32 * i] : 0.0f;
    const float ks = c.k_scales[kvh * (c.capacity / c.block) + j / c.block];
    for (int t = max(0, j - held); t < rows; ++t)
        for (int g = 0; g < group; ++g) {
            const int64_t row = static_cast<int64_t>(b) * a.rows_per_seq + t;
            const int head = h * group + g;
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < kDims; ++i)
                if (lane + 32 * i < d) s = fmaf(a.q[row * a.q_stride + head * d + lane + 32 * i], k[i], s);
            for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            sum += expf(s * ks * a.scale - lse[row * a.heads + head]);
        }
    if (lane == 0) c.weights[kvh * c.capacity + j] += sum;
}

}  // namespace

size_t kv8_attention_bytes(int32_t batch, int32_t rows_per_seq, int32_t heads, int32_t, int32_t, int32_t) {
    return static_cast<size_t>(batch) * rows_per_seq * heads * sizeof(float);
}

cudaError_t launch_kv8_attention(const Kv8Attention& a, int, cudaStream_t s) {
    const Kv8& c = a.cache;
    float* lse = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + kv8_counter_bytes(c.batch, c.kv_heads));
    cudaError_t e = launch_dependent(kv8_attention_rows_kernel, dim3(a.rows_per_seq, a.heads, c.batch),
                                     dim3(kWarps * 32), 0, s, a, lse);
    if (e == cudaSuccess && a.accumulate)
        e = launch_dependent(kv8_weights_kernel, dim3((c.capacity + kWarps - 1) / kWarps, c.kv_heads, c.batch),
                             dim3(kWarps * 32), 0, s, a, lse);
    return e;
}

}  // namespace kt
