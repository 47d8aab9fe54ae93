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
constexpr uint32_t kTiny = 0x0d800000u;  // bits of 2^-100
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
// The nearest integer to y, ties to even, in the low bits: adding 1.5 x 2^23 rounds.
// (A scalar operation: the assembler contracts packed products and sums into one
// rounding.)  A code's y stays below 127.5: its three roundings are 2^-24 each.
__device__ __forceinline__ uint32_t nearest_bits(float y) { return __float_as_uint(__fadd_rn(y, 12582912.0f)); }
__device__ __forceinline__ uint32_t code_bits(float x, float inverse) { return nearest_bits(__fmul_rn(x, inverse)); }
__device__ __forceinline__ uint32_t codes_of(float4 x, float inverse) {
    if (inverse == 0.0f) return 0;  // NaN and infinity times 0 are not 0
    const uint32_t lo = dev::prmt(code_bits(x.x, inverse), code_bits(x.y, inverse), 0x0040);
    const uint32_t hi = dev::prmt(code_bits(x.z, inverse), code_bits(x.w, inverse), 0x0040);
    return dev::prmt(lo, hi, 0x5410);
}
// Two products at a time.
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ uint64_t pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
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
    if (aligned) return __ldg(reinterpret_cast<const float4*>(p));
    return make_float4(p[0], p[1], p[2], p[3]);
}

// One CTA per (block that the new tokens touch, head, sequence, key or value).
// kColumns threads (a power of two, head_dim / 4 or more) share a slot, four values
// each, so no index needs a division; a block's values stay in registers between the
// search for the largest and their rounding, each read once.  The CTA of a sequence's
// first touched block is the only one that reads the old tail and writes the new one.
// Bound by memory: every value is read as it is, in fp32, and leaves as a byte.  4 prompts
// of 1021 tokens, 8 heads of 128: 12.1 us, 43.7 MB, 3.6 TB/s; a token of each of 64
// sequences, whose blocks' tails are read again: 8.2 us, 33.6 MB, 4.1 TB/s.  (With index
// divisions and one value a thread 19.7 and 16.4 us.)
template <int kColumns>
__global__ void __launch_bounds__(kThreads) kv8_store_kernel(Kv8 c, const float* __restrict__ k,
                                                             const float* __restrict__ v, int64_t k_stride,
                                                             int64_t v_stride, int aligned, int rows_per_seq,
                                                             const int32_t* __restrict__ counts,
                                                             int32_t* __restrict__ status) {
    constexpr int kSlots = kThreads / kColumns, kVecs = 64 / kSlots;  // slots a pass, passes of the largest block
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
    const int shift = 31 - __clz(c.block), first = held >> shift, inside = held - (first << shift);
    if (n == 0 || (x << shift) >= inside + n) return;
    const int64_t head = static_cast<int64_t>(b) * c.kv_heads + h;
    const int col = threadIdx.x % kColumns * 4, slot0 = threadIdx.x / kColumns;
    const bool has = col < c.head_dim;
    int8_t* codes = (value ? c.v_codes : c.k_codes) +
                    (head * c.capacity + (static_cast<int64_t>(first + x) << shift)) * c.head_dim + col;
    float* tail = (value ? c.v_tail : c.k_tail) + (head << shift) * c.head_dim + col;
    const int64_t stride = value ? v_stride : k_stride;
    const float* rows = (value ? v : k) + static_cast<int64_t>(b) * rows_per_seq * stride + h * c.head_dim + col;
    const int row0 = (x << shift) - inside + slot0;  // negative: a slot that was held before (x == 0)

    float4 r[kVecs];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int slot = slot0 + i * kSlots, row = row0 + i * kSlots;
        r[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (has && slot < c.block && row < n)
            r[i] = row < 0 ? *reinterpret_cast<const float4*>(tail + slot * c.head_dim) : load4(rows + row * stride, aligned);
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) top = max(top, magnitude(r[i]));
    const BlockScale s = block_scale(block_max(top));
    if (threadIdx.x == 0) (value ? c.v_scales : c.k_scales)[head * (c.capacity >> shift) + first + x] = s.scale;
    const int last = (held + n) >> shift;  // the new open block
    const bool grows = x == 0 && last == first;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int slot = slot0 + i * kSlots, row = row0 + i * kSlots;
        if (!has || slot >= c.block || row >= n) continue;
        *reinterpret_cast<uint32_t*>(codes + slot * c.head_dim) = codes_of(r[i], s.inverse);
        if (grows && row >= 0) *reinterpret_cast<float4*>(tail + slot * c.head_dim) = r[i];
    }
    if (x == 0 && last != first && has) {  // the rows left over after the last full block
        const int left = held + n - (last << shift);
        for (int slot = slot0; slot < left; slot += kSlots)
            *reinterpret_cast<float4*>(tail + slot * c.head_dim) = load4(rows + (n - left + slot) * stride, aligned);
    }
    if (c.weights != nullptr && !value && threadIdx.x < c.block) {
        const int row = (x << shift) - inside + threadIdx.x;
        if (row >= 0 && row < n) c.weights[head * c.capacity + held + row] = 0.0f;
    }
}

// RoPE (RoPE.kt:117-155) of the query and key heads of fused q|k|v rows in place: a
// thread has a pair (i, i + half) of one head.
__global__ void __launch_bounds__(kThreads) rope_seqs_kernel(float* __restrict__ qkv, int heads, int head_dim, int64_t stride,
                                                             const float* __restrict__ inv_freq,
                                                             const int32_t* __restrict__ position, int rows_per_seq) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const int half = head_dim / 2, r = blockIdx.y, at = *position + r % rows_per_seq;
    float* row = qkv + r * stride;
    for (int e = blockIdx.x * kThreads + threadIdx.x; e < heads * half; e += gridDim.x * kThreads) {
        const int head = e / half, i = e - head * half;
        float* v = row + head * head_dim;
        float sn, cs;
        sincosf(static_cast<float>(at) * inv_freq[i], &sn, &cs);
        const float x1 = v[i], x2 = v[i + half];
        v[i] = x1 * cs - x2 * sn;
        v[i + half] = x1 * sn + x2 * cs;
    }
}

__global__ void kv8_advance_kernel(int32_t* __restrict__ lengths, int batch, int rows,
                                   const int32_t* __restrict__ counts, int limit) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    for (int b = threadIdx.x; b < batch; b += blockDim.x) {
        // what the store of these rows added
        const int64_t to = static_cast<int64_t>(lengths[b]) + kv8_rows(counts, b, rows);
        lengths[b] = static_cast<int32_t>(min(max(to, static_cast<int64_t>(0)), static_cast<int64_t>(limit)));
    }
}

// ------------------------------------------------------------ eviction

constexpr int kSelectThreads = 1024;
constexpr int kSelectEach = 8;  // slots of a chunk a thread holds
constexpr int kBins = 2048;

// Weights ordered as unsigned integers: negative ones reversed below the others,
// -0 as 0, NaN above all.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Exclusive prefix sum of v over the block's threads, and the sum of all; barriers on both sides.
__device__ __forceinline__ int block_prefix(int v, int& all) {
    __shared__ int part[kSelectThreads / 32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int upto = v;
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
    }
    __syncthreads();
    if (lane == 31) part[warp] = upto;
    __syncthreads();
    int before = part[lane];
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += u;
    }
    all = __shfl_sync(0xffffffffu, before, 31);
    before = __shfl_sync(0xffffffffu, before, max(warp - 1, 0));
    return upto - v + (warp > 0 ? before : 0);
}

// One CTA per (head, sequence).  The smallest key that is kept comes from three
// counting passes over its digits of 11, 11 and 10 bits (integer counts: any order of
// the atomics gives the same), then the kept slots go in order into `order` and their
// weights to the front.  Latency-bound: the weights are read from L1 after the first
// pass.  A head of 6401 slots takes 10.5 us, 3.9 of them the first pass and 3.1 the
// last; one of 62 slots 6 us.  (Bit by bit, 16 sequences x 8 heads of 8k took 58 us.)
__global__ void __launch_bounds__(kSelectThreads) kv8_select_kernel(Kv8 c, int keep, int recent,
                                                                    int32_t* __restrict__ order) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    __shared__ int bins[kBins];
    __shared__ uint32_t found;  // the digit, and how many above it
    __shared__ int above_found;
    const int b = blockIdx.y, h = blockIdx.x, held = kv8_held(c, b);
    if (held <= keep) return;
    const int64_t head = static_cast<int64_t>(b) * c.kv_heads + h;
    float* w = c.weights + head * c.capacity;
    order += head * c.capacity;
    const int candidates = held - recent;
    uint32_t bound = 0;         // the key's digits found so far
    int want = keep - recent;   // how many to keep among the candidates that share them
    if (want > 0) {
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int low = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
            const uint32_t digits = (1u << width) - 1, above_mask = pass == 0 ? 0u : ~0u << (low + width);
            for (int i = threadIdx.x; i < kBins; i += kSelectThreads) bins[i] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < candidates; i += kSelectThreads) {
                const uint32_t key = order_key(w[i]);
                if ((key & above_mask) == bound) atomicAdd(bins + (key >> low & digits), 1);
            }
            __syncthreads();
            // from the top: thread i has bins kBins - 2 - 2 i and the one above it
            const int hi = kBins - 1 - 2 * threadIdx.x, n1 = bins[hi], n0 = bins[hi - 1];
            int all;
            const int before = block_prefix(n1 + n0, all);
            if (before < want && before + n1 + n0 >= want) {
                const bool upper = before + n1 >= want;
                found = upper ? hi : hi - 1;
                above_found = upper ? before : before + n1;
            }
            __syncthreads();
            bound |= found << low;
            want -= above_found;
            __syncthreads();
        }
    } else {
        bound = 0xffffffffu;  // none; a NaN's key is not above it, and no tie is wanted
    }
    // `want` is now how many of those equal to the bound are kept, lowest slots first.  A warp
    // has 32 kSelectEach slots of a chunk, a lane every 32nd, so loads and stores run along the
    // slots; slots kept for certain and ties before a slot are counted together, in halves of a word.
    const int lane = threadIdx.x % 32, first = threadIdx.x / 32 * (32 * kSelectEach) + lane;
    int kept_before = 0, tied_before = 0;
    for (int base = 0; base < held; base += kSelectThreads * kSelectEach) {
        float x[kSelectEach];
        uint32_t certain[kSelectEach], tied[kSelectEach];  // the warp's slots
        int counts = 0;
#pragma unroll
        for (int j = 0; j < kSelectEach; ++j) {
            const int i = base + first + 32 * j;
            certain[j] = tied[j] = 0;
            if (i - lane >= held) continue;
            x[j] = i < held ? w[i] : 0.0f;
            const uint32_t key = order_key(x[j]);
            certain[j] = __ballot_sync(0xffffffffu, i < held && (i >= candidates || key > bound));
            tied[j] = __ballot_sync(0xffffffffu, i < candidates && key == bound);
            counts += __popc(certain[j]) + (__popc(tied[j]) << 16);
        }
        int all;
        const int before = block_prefix(lane == 0 ? counts : 0, all);  // (every weight of the chunk has been read)
        const int warp_before = __shfl_sync(0xffffffffu, before, 0);
        int sure = kept_before + (warp_before & 0xffff), ties = tied_before + (warp_before >> 16);
#pragma unroll
        for (int j = 0; j < kSelectEach; ++j) {
            if ((certain[j] | tied[j]) == 0) continue;
            const uint32_t below = (1u << lane) - 1;
            const int rank = ties + __popc(tied[j] & below);
            if ((certain[j] >> lane & 1) || ((tied[j] >> lane & 1) && rank < want)) {
                // at most the slot itself: later chunks lose nothing
                const int place = sure + __popc(certain[j] & below) + min(rank, want);
                order[place] = base + first + 32 * j;
                w[place] = x[j];
            }
            sure += __popc(certain[j]);
            ties += __popc(tied[j]);
        }
        kept_before += all & 0xffff;
        tied_before += all >> 16;
    }
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
// 16 bytes global -> shared, asynchronously; zeros unless `real`.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
// A warp moves a unit of 64 tokens: lane l has piece l % kPieces (16 codes) of every
// (32 / kPieces)-th token, all in registers at once.  A cluster of CTAs walks the
// units of one (head, sequence, key or value) in rounds, a unit to each of its warps:
// the token that moves to slot i comes from a slot >= i, so what a round overwrites no
// later round still needs, and a round's own codes have been read at the barrier ahead
// of its writes.  For the same reason the next unit's codes may come by asynchronous
// copies while this one is quantised.  The barrier's arrival is a release, so that every
// code read before it is read before what others write after it; it comes once the last
// round's writes, which it also waits for, are long under way (16 sequences x 8 heads
// with selection: 87 us, ahead of the search for the largest 89, with a relaxed arrival,
// which promises no order, 85, events around cold calls).  Where there are few heads, a cluster of up to 8 CTAs
// shares each.  16 sequences x 8 heads of 128, 4000 of 8k slots kept: 68 us for 262 MB,
// 3.9 TB/s; about 9 instructions a code, issued in 55% of the cycles.  (With the relaxed
// arrival 65; from there, without the copies ahead 84 us, with five CTAs on an SM, whose
// registers spill, 77.)
constexpr int kUnit = 64;
constexpr int kMoveWarps = 4;
template <int kPieces>
struct MoveShape {
    static constexpr int kTokens = 32 / kPieces, kLoads = kUnit / kTokens, kPer16 = 16 / kTokens;
    static constexpr int kBuffer = kLoads * 32 * 16;  // bytes of a warp: [load][lane]
    static constexpr int kSmem = kMoveWarps * kBuffer;
};
template <int kPieces>
__global__ void __launch_bounds__(kMoveWarps * 32, 4) kv8_move_kernel(Kv8 c, int keep, const int32_t* __restrict__ order) {
    using S = MoveShape<kPieces>;
    constexpr int kTokens = S::kTokens, kLoads = S::kLoads, kPer16 = S::kPer16;
    extern __shared__ __align__(16) unsigned char move_smem[];
    __shared__ int from_of[kMoveWarps][kUnit];
    __shared__ float scale_of[2][kMoveWarps][kUnit];
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const int b = blockIdx.z >> 1, h = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const bool value = blockIdx.z & 1;
    if (kv8_held(c, b) <= keep) return;
    const int64_t head = static_cast<int64_t>(b) * c.kv_heads + h;
    order += head * c.capacity;
    const int shift = 31 - __clz(c.block), d = c.head_dim, col = lane % kPieces * 16, token0 = lane / kPieces;
    const bool has = col < d;
    int8_t* codes = (value ? c.v_codes : c.k_codes) + head * c.capacity * d + col;
    float* scales = (value ? c.v_scales : c.k_scales) + head * (c.capacity >> shift);
    float* tail = (value ? c.v_tail : c.k_tail) + (head << shift) * d + col;
    const int full = keep >> shift << shift;  // slots of whole blocks
    const uint32_t buffer = dev::smem_u32(move_smem) + warp * S::kBuffer + lane * 16;
    const int stride = gridDim.x * kMoveWarps * kUnit;
    int next[2];  // the slots that move to lane and lane + 32 of the unit after
    auto look = [&](int base) {
#pragma unroll
        for (int i = 0; i < 2; ++i) next[i] = base + 32 * i + lane < keep ? order[base + 32 * i + lane] : -1;
    };
    // Asynchronous copies of the unit whose slots are in `next`; its scales to half y of scale_of.
    auto fetch = [&](int y) {
        __syncwarp();  // the last unit's tokens have been used
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            from_of[warp][32 * i + lane] = next[i];
            scale_of[y][warp][32 * i + lane] = next[i] >= 0 ? scales[next[i] >> shift] : 0.0f;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int f = from_of[warp][token0 + i * kTokens];
            const bool real = f >= 0 && has;
            copy16(buffer + i * 512, codes + (real ? static_cast<int64_t>(f) * d : 0), real);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // A packed sum, of a product by a one that the assembler does not know: it would join
    // a packed sum with the product before it, in one rounding.
    float one = 1.0f;
    asm volatile("" : "+f"(one));
    const uint64_t ones = pair(one, one), magic = pair(12582912.0f, 12582912.0f);
    int base = (blockIdx.x * kMoveWarps + warp) * kUnit, y = 0;
    look(base);
    fetch(0);
    look(base + stride);
    for (int left = (keep + kUnit - 1) / kUnit; left > 0; left -= gridDim.x * kMoveWarps, base += stride, y ^= 1) {
        const float* const scale = scale_of[y][warp] + token0;
        uint4 r[kLoads];
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int i = 0; i < kLoads; ++i) r[i] = lds128(buffer + i * 512);
        // the largest value of each 16 tokens: scale x largest code, exactly the largest product
        uint32_t top[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t words[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
            uint32_t most = 0, least = 0;  // signed 16-bit lanes; a code is a lane's high byte, what is below it does not matter
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                most = __vimax3_s16x2(most, words[j], words[j] << 8);
                least = __vimin3_s16x2(least, words[j], words[j] << 8);
            }
            const int hi = max(static_cast<int>(most) >> 24, static_cast<int8_t>(most >> 8));
            const int lo = -min(static_cast<int>(least) >> 24, static_cast<int8_t>(least >> 8));
            const float m = static_cast<float>(max(hi, lo));
            top[i / kPer16] = max(top[i / kPer16], magnitude(__fmul_rn(scale[i * kTokens], m)));
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        if (left > gridDim.x * kMoveWarps) {  // the codes are in registers
            fetch(y ^ 1);
            look(base + 2 * stride);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) top[g] = __reduce_max_sync(0xffffffffu, top[g]);
        if (shift >= 5) top[0] = top[1] = max(top[0], top[1]), top[2] = top[3] = max(top[2], top[3]);
        if (shift >= 6) top[0] = top[1] = top[2] = top[3] = max(top[0], top[2]);
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const BlockScale bs = block_scale(top[g]);
            top[g] = __float_as_uint(bs.inverse);
            const int slot = base + 16 * g;
            if (lane == 0 && slot < keep && (slot & (c.block - 1)) == 0) scales[slot >> shift] = bs.scale;
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int slot = base + token0 + i * kTokens;
            if (!has || slot >= keep) continue;
            uint32_t words[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
            // converted again: kept from the search, the floats would not fit the registers
            asm volatile("" : "+r"(words[0]), "+r"(words[1]), "+r"(words[2]), "+r"(words[3]));
            const float inverse = __uint_as_float(top[i / kPer16]), s = scale[i * kTokens];
            uint32_t out[4];
            const uint64_t ss = pair(s, s), ii = pair(inverse, inverse);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint64_t x0 = mul2(ss, pair(static_cast<float>(static_cast<int8_t>(words[j])),
                                                  static_cast<float>(static_cast<int8_t>(words[j] >> 8))));
                const uint64_t x1 = mul2(ss, pair(static_cast<float>(static_cast<int8_t>(words[j] >> 16)),
                                                  static_cast<float>(static_cast<int8_t>(words[j] >> 24))));
                const float2 y0 = unpair(fma2(mul2(x0, ii), ones, magic)), y1 = unpair(fma2(mul2(x1, ii), ones, magic));
                const uint32_t lo = dev::prmt(__float_as_uint(y0.x), __float_as_uint(y0.y), 0x0040);
                const uint32_t hi = dev::prmt(__float_as_uint(y1.x), __float_as_uint(y1.y), 0x0040);
                out[j] = dev::prmt(lo, hi, 0x5410);
                if (slot >= full) {
                    const float2 a = unpair(x0), e = unpair(x1);
                    *reinterpret_cast<float4*>(tail + static_cast<int64_t>(slot - full) * d + 4 * j) = make_float4(a.x, a.y, e.x, e.y);
                }
            }
            if (inverse == 0.0f) out[0] = out[1] = out[2] = out[3] = 0;
            *reinterpret_cast<uint4*>(codes + static_cast<int64_t>(slot) * d) = make_uint4(out[0], out[1], out[2], out[3]);
        }
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
    if (!aligned16(c->k_codes) || !aligned16(c->v_codes) || !aligned16(c->k_tail) || !aligned16(c->v_tail))
        return "codes and tails must be 16-byte aligned";
    return nullptr;
}

}  // namespace kt

using namespace kt;

kt_status kt_rope_seqs(kt_ctx* ctx, float* qkv, int32_t rows, int32_t q_width, int32_t kv_heads, int32_t head_dim,
                       const float* inv_freq, const int32_t* position, int32_t rows_per_seq, void* stream) {
    if (!ctx || !qkv || !inv_freq || !position || rows <= 0 || rows > 65535 || head_dim <= 0 || head_dim % 2 != 0 ||
        q_width % head_dim != 0 || kv_heads <= 0 || rows_per_seq <= 0 || rows % rows_per_seq != 0)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "bad rope_seqs arguments");
    return c_entry(ctx, [&] {
        const int heads = q_width / head_dim + kv_heads;
        const dim3 grid((heads * (head_dim / 2) + kThreads - 1) / kThreads, rows);
        return entry_launch(launch_dependent(rope_seqs_kernel, grid, dim3(kThreads), 0, static_cast<cudaStream_t>(stream), qkv,
                                             heads, head_dim, static_cast<int64_t>(q_width) + 2ll * kv_heads * head_dim,
                                             inv_freq, position, rows_per_seq),
                            "rope_seqs launch");
    });
}

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
        // blocks that rows can touch from any place in the first
        const dim3 grid((rows + cache->block - 2) / cache->block + 1, cache->kv_heads, 2 * cache->batch);
        const auto kernel = cache->head_dim > 64 ? kv8_store_kernel<32> : cache->head_dim > 32 ? kv8_store_kernel<16> : kv8_store_kernel<8>;
        return entry_launch(launch_dependent(kernel, grid, dim3(kThreads), 0, static_cast<cudaStream_t>(stream), *cache, k, v,
                                             k_stride, v_stride, aligned, rows_per_seq, counts, status),
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
    if (batch < 1 || limit < 0 || (counts && rows < 0)) return entry_fail(KT_ERR_INVALID_ARGUMENT, "bad advance arguments");
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
        if (e == cudaSuccess) {
            // CTAs that share a head's units: while one to a head leaves SMs idle and there
            // are units for more
            const int64_t alone = 2ll * cache->batch * cache->kv_heads;
            const int units = (keep + kUnit - 1) / kUnit;
            int share = 1;
            while (share < 8 && alone * share * 2 <= 8ll * ctx->sm_count && units > share * kMoveWarps) share *= 2;
            const auto kernel = cache->head_dim > 64 ? kv8_move_kernel<8> : cache->head_dim > 32 ? kv8_move_kernel<4> : kv8_move_kernel<2>;
            cudaLaunchConfig_t lc = {};
            lc.gridDim = dim3(share, cache->kv_heads, 2 * cache->batch);
            lc.blockDim = dim3(kMoveWarps * 32);
            lc.dynamicSmemBytes = cache->head_dim > 64 ? MoveShape<8>::kSmem : cache->head_dim > 32 ? MoveShape<4>::kSmem : MoveShape<2>::kSmem;
            lc.stream = s;
            cudaLaunchAttribute attr[2];
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[0].val.programmaticStreamSerializationAllowed = 1;
            attr[1].id = cudaLaunchAttributeClusterDimension;
            attr[1].val.clusterDim.x = share;
            attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
            lc.attrs = attr;
            lc.numAttrs = 2;
            e = cudaLaunchKernelEx(&lc, kernel, static_cast<Kv8>(*cache), keep, static_cast<const int32_t*>(order));
        }
        return entry_launch(e, "kv8 evict launch");
    });
}
