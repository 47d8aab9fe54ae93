// kt_paged.h -- the paged 16-bit key/value cache as its kernels see it, the list of
// tiles that its attention kernels share out, and their launchers (kt_paged.cu,
// kt_paged_attention.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kt_kv8.h"  // c_entry, launch_dependent, allow_shared

namespace kt {

using Paged = kt_paged_cache;  // passed to kernels by value

// Scratch layout (kt_paged_scratch_bytes): a counter for each CTA of the kernel of few
// vectors, zero between calls; the items that the kernel of many vectors has cut; the parts
// of cut items, two for each CTA.
constexpr size_t kPagedCounterBytes = 4096;  // (include/kt_cuda.h and paged.py give this number)
constexpr size_t kPagedCutBytes = 8192, kPagedPartsAt = kPagedCounterBytes + kPagedCutBytes;
constexpr int kPagedRowsCtas = 512, kPagedManyCtas = 256;  // of a launch, at most
static_assert(kPagedRowsCtas * sizeof(int32_t) <= kPagedCounterBytes, "a counter each");

struct PagedAttention {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* counts;    // NULL: rows everywhere
    const uint32_t* visible;  // NULL: row t sees the new tokens 0..t
    const void* q;
    void* out;
    void* scratch;
    int64_t q_stride;
    int32_t batch, kv_heads, head_dim, pages, page_shift, table_stride, capacity;
    int32_t rows, heads, group, words;  // rows of a sequence, words of a row of `visible`
    float factor;                       // scale * log2(e)
    int32_t out_f32, aligned;           // aligned to 16 bytes: bit 0 the rows of q, bit 1 out
};
// Boxes of the tensor maps: 64 dims of the slots of a page, at most 64 of them.
constexpr int kPagedBox = 64;
// Which kernel runs, and its launch (kt_paged_attention.cu); the kernel of many vectors
// (kt_paged_many.cu).
cudaError_t launch_paged_attention(const Paged& c, int layer, const PagedAttention& a, int sm_count, int32_t* err,
                                   cudaStream_t s);
cudaError_t launch_paged_many(bool bf16, const CUtensorMap (&maps)[2], const PagedAttention& a, int sm_count, int32_t* err,
                              cudaStream_t s);
size_t paged_rows_bytes();
size_t paged_many_bytes(int sm_count);

#ifdef __CUDACC__
namespace paged {

// Tokens that sequence b holds, and rows of this call that are tokens, whatever the
// caller left in the arrays.
__device__ __forceinline__ int held_of(const int32_t* lengths, int b, int capacity) {
    return min(max(lengths[b], 0), capacity);
}
__device__ __forceinline__ int rows_of(const int32_t* counts, int b, int rows) {
    return counts == nullptr ? rows : min(max(counts[b], 0), rows);
}

// Zeros for the rows that are no tokens; by one warp of every CTA.
__device__ __forceinline__ void zero_rows(const PagedAttention& a) {
    const int lane = threadIdx.x % 32, width = a.heads * a.head_dim;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.rows;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * 32; r0 < rows; r0 += static_cast<int64_t>(gridDim.x) * 32) {
        bool token = true;
        if (r0 + lane < rows) {
            const int b = static_cast<int>((r0 + lane) / a.rows), t = static_cast<int>((r0 + lane) % a.rows);
            token = t < min(rows_of(a.counts, b, a.rows), a.capacity - held_of(a.lengths, b, a.capacity));
        }
        for (uint32_t none = __ballot_sync(0xffffffffu, !token); none != 0; none &= none - 1) {
            const int64_t at = (r0 + __ffs(none) - 1) * width;
            for (int i = lane; i < width; i += 32) {
                if (a.out_f32) static_cast<float*>(a.out)[at + i] = 0.0f;
                else static_cast<uint16_t*>(a.out)[at + i] = 0;
            }
        }
    }
}
// Where the query and the result of an item's vector begin.
__device__ __forceinline__ int64_t place_of(const PagedAttention& a, int b, int head, int v, int64_t stride) {
    const int row = v / a.group;
    return (static_cast<int64_t>(b) * a.rows + row) * stride + static_cast<int64_t>(head * a.group + v - row * a.group) * a.head_dim;
}

// A place in a ring of kUnits, and the phase of its barrier.
template <int kUnits>
struct Ring {
    int at = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++at == kUnits) at = 0, phase ^= 1;
    }
};
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {  // of numbers that are not negative
    return (x | y) >> 32 == 0 ? static_cast<int64_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(y)) : x / y;
}

// An item of the attention's work: kVectors query vectors (rows x heads of a group, in
// row order) of one sequence and key/value head, over tiles of kTile slots.
struct Item {
    int64_t base;            // index of the item's first unit in the list of all
    int entry;               // sequence * vector tiles + vector tile
    int b, head, v0, valid;  // first vector, how many there are
    int held, count;         // tokens held, rows that are tokens
    int sees, tiles;         // slots the last vector sees
    int from, to;            // tiles of this CTA
    int last;                // the CTA's last item
};
// How the list of all tiles is shared out, and each warp's place in its CTA's run.  In
// shared memory: the loops over tiles need their registers.
template <int kWarps>
struct Plan {
    int64_t share, spare, begin, end;
    int64_t sums[kWarps], items[kWarps], base;
    int entry, dealt;
    Item at[kWarps];
};

// The list of all tiles, sequences first, then vector tiles, then heads; an item is kStart
// units, what entering it costs, and one for each tile.  Equal runs of units go to the
// CTAs: ragged batches, single long sequences and the triangle of a prompt load every SM
// alike.  Lengths are read here, on the device, so a captured launch fits any.
//
// With kDeal, equal sequences of several vector tiles (a prompt) are not cut where there are
// kDeal items or more to a CTA: they are dealt out whole, the longest first, every other
// round backwards, so that the sums are as equal and nothing has to be merged.
template <int kWarps, int kVectors, int kTile, int kStart, int kLeast, int kWhole, int kDeal>
struct WorkList {
    const PagedAttention& a;
    Plan<kWarps>& plan;

    __device__ __forceinline__ int vector_tiles() const { return (a.rows * a.group + kVectors - 1) / kVectors; }
    __device__ __forceinline__ void load(Item& it, int entry, int vts) const {  // all but head, base and the tiles
        it.entry = entry;
        it.b = entry / vts;
        it.v0 = (entry - it.b * vts) * kVectors;
        it.held = held_of(a.lengths, it.b, a.capacity);
        it.count = min(rows_of(a.counts, it.b, a.rows), a.capacity - it.held);
        it.valid = min(kVectors, it.count * a.group - it.v0);
        it.sees = it.valid <= 0 ? 0 : a.visible ? it.held + it.count : it.held + (it.v0 + it.valid - 1) / a.group + 1;
        it.tiles = (it.sees + kTile - 1) / kTile;
    }
    // Item `rank` of those dealt, the last vector tile's first: by the item's round and this CTA.
    __device__ bool deal(Item& it, int64_t round, int vts) const {
        const int64_t among = static_cast<int64_t>(a.batch) * a.kv_heads, all = among * vts;
        const int64_t rank = round * gridDim.x + (round % 2 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        if (rank >= all) return false;
        const int vt = vts - 1 - static_cast<int>(rank / among), which = static_cast<int>(rank % among);
        load(it, which / a.kv_heads * vts + vt, vts);
        it.head = which % a.kv_heads;
        it.base = round;
        it.from = 0, it.to = it.tiles;
        // (the next round's item of this CTA, if there is one)
        const int64_t next = (round + 1) * gridDim.x + (round % 2 ? blockIdx.x : gridDim.x - 1 - blockIdx.x);
        it.last = next >= all;
        return true;
    }
    __device__ __forceinline__ void cut(Item& it) const {
        it.from = static_cast<int>(max(static_cast<int64_t>(0), plan.begin - it.base - kStart));
        it.to = static_cast<int>(min(static_cast<int64_t>(it.tiles), max(static_cast<int64_t>(0), plan.end - it.base - kStart)));
        it.last = it.base + it.tiles + kStart >= plan.end;
    }
    __device__ int cta_of(int64_t unit) const {  // the CTA whose run holds it
        const int64_t longer = plan.spare * (plan.share + 1);
        return static_cast<int>(unit < longer ? quotient(unit, plan.share + 1) : plan.spare + quotient(unit - longer, plan.share));
    }
    // The CTAs that share an item's tiles are first_cta .. last_cta.
    __device__ int first_cta(const Item& it) const { return cta_of(it.base + kStart); }
    __device__ int last_cta(const Item& it) const { return cta_of(it.base + kStart + it.tiles - 1); }

    // By all threads of the CTA: shares out the list; false: nothing for this CTA.  A CTA gets
    // at least kLeast tiles or an item; items of at most kWhole tiles are not cut for more CTAs.
    __device__ bool start() const {
        constexpr int kThreads = kWarps * 32;
        const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, vts = vector_tiles();
        if (kDeal > 0 && vts > 1 && static_cast<int64_t>(a.batch) * a.kv_heads * vts >= static_cast<int64_t>(kDeal) * gridDim.x) {
            bool equal = true;
            for (int b = threadIdx.x; b < a.batch; b += kThreads)
                equal = equal && a.lengths[b] == a.lengths[0] && (a.counts == nullptr || a.counts[b] == a.counts[0]);
            if (__syncthreads_and(equal)) {
                if (threadIdx.x == 0) plan.dealt = 1;
                Item it;
                const bool any = deal(it, 0, vts);
                if (lane == 0) plan.at[warp] = it;
                __syncthreads();
                return any;
            }
        }
        const int entries = a.batch * vts, each = (entries + kThreads - 1) / kThreads;
        if (entries <= 32) {  // an entry to a lane, every warp for itself (the sums of all threads took 1 us longer)
            Item it;
            it.tiles = 0;
            if (lane < entries) load(it, lane, vts);
            const int64_t units = it.tiles > 0 ? static_cast<int64_t>(it.tiles + kStart) * a.kv_heads : 0;
            const int64_t items = static_cast<int64_t>(__popc(__ballot_sync(0xffffffffu, it.tiles > 0))) * a.kv_heads;
            const bool whole = !__any_sync(0xffffffffu, it.tiles > kWhole);
            int64_t upto = units;
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const int64_t total = __shfl_sync(0xffffffffu, upto, 31);
            if (items == 0) return false;
            const int64_t ctas = min(static_cast<int64_t>(gridDim.x), whole ? items : max(items, quotient(total - items * kStart, kLeast)));
            if (blockIdx.x >= ctas) return false;
            const int64_t share = quotient(total, ctas), spare = total - share * ctas;
            const int64_t begin = blockIdx.x * share + min(static_cast<int64_t>(blockIdx.x), spare);
            if (lane == __ffs(__ballot_sync(0xffffffffu, upto > begin)) - 1) {  // (equal numbers from every warp)
                plan.share = share, plan.spare = spare, plan.begin = begin;
                plan.end = begin + share + (blockIdx.x < spare);
                plan.dealt = 0;
                it.head = static_cast<int>(quotient(begin - (upto - units), it.tiles + kStart));
                it.base = upto - units + static_cast<int64_t>(it.head) * (it.tiles + kStart);
                cut(it);
                plan.at[warp] = it;
            }
            __syncthreads();
            return true;
        }
        if (threadIdx.x == 0) plan.dealt = 0;
        const int from = min(entries, static_cast<int>(threadIdx.x) * each), to = min(entries, from + each);
        Item it;
        int64_t units = 0, items = 0;
        int longest = 0;
        for (int e = from; e < to; ++e) {
            load(it, e, vts);
            if (it.tiles > 0) units += it.tiles + kStart, ++items;
            longest = max(longest, it.tiles);
        }
        units *= a.kv_heads, items *= a.kv_heads;
        int64_t upto = units;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        for (int o = 16; o > 0; o >>= 1) items += __shfl_xor_sync(0xffffffffu, items, o);
        if (lane == 31) plan.sums[warp] = upto, plan.items[warp] = items;
        const bool whole = !__syncthreads_or(longest > kWhole);
        int64_t before = upto - units, total = 0;
        items = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += plan.sums[w];
            total += plan.sums[w];
            items += plan.items[w];
        }
        if (items == 0) return false;
        const int64_t ctas = min(static_cast<int64_t>(gridDim.x), whole ? items : max(items, quotient(total - items * kStart, kLeast)));
        if (blockIdx.x >= ctas) return false;
        const int64_t share = quotient(total, ctas), spare = total - share * ctas;
        const int64_t begin = blockIdx.x * share + min(static_cast<int64_t>(blockIdx.x), spare);
        if (threadIdx.x == 0) {
            plan.share = share, plan.spare = spare, plan.begin = begin;
            plan.end = begin + share + (blockIdx.x < spare);
        }
        if (before <= begin && begin < before + units) {  // one thread
            for (int e = from; e < to; ++e) {
                load(it, e, vts);
                const int64_t n = it.tiles > 0 ? static_cast<int64_t>(it.tiles + kStart) * a.kv_heads : 0;
                if (begin < before + n) {
                    plan.entry = e;
                    plan.base = before;
                    break;
                }
                before += n;
            }
        }
        __syncthreads();
        if (lane == 0) {
            Item& mine = plan.at[warp];
            load(it, plan.entry, vts);
            it.head = static_cast<int>(quotient(begin - plan.base, it.tiles + kStart));
            it.base = plan.base + static_cast<int64_t>(it.head) * (it.tiles + kStart);
            cut(it);
            mine = it;
        }
        __syncwarp();
        return true;
    }
    // To the warp's next item; by its lane 0.
    __device__ void step() const {
        Item it = plan.at[threadIdx.x / 32];
        if (kDeal > 0 && plan.dealt) {
            deal(it, it.base + 1, vector_tiles());
            plan.at[threadIdx.x / 32] = it;
            return;
        }
        const int64_t base = it.base + it.tiles + kStart;
        if (++it.head == a.kv_heads) {
            it.head = 0;
            const int vts = vector_tiles();
            do load(it, it.entry + 1, vts);
            while (it.tiles == 0);  // (units are left, so a later entry has tiles)
        }
        it.base = base;
        cut(it);
        plan.at[threadIdx.x / 32] = it;
    }
    // The same by the whole warp; false: the run ends before it.
    __device__ __forceinline__ bool next() const {
        if (plan.at[threadIdx.x / 32].last) return false;
        __syncwarp();
        if (threadIdx.x % 32 == 0) step();
        __syncwarp();
        return true;
    }
};

// Which of `n` (at most 32) slots from `slot` on row t sees: bit i for slot + i.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t seen_bits(const PagedAttention& a, const Item& it, int t, int slot) {
    if (a.visible == nullptr) return low_bits(min(it.held + t + 1, it.held + it.count) - slot);
    uint32_t bits = low_bits(it.held - slot);
    const int u = slot - it.held;  // the new token in `slot`
    if (u > -32 && u < it.count) {
        const uint32_t* row = a.visible + (static_cast<int64_t>(it.b) * a.rows + t) * a.words;
        uint32_t fresh;
        if (u < 0) {
            fresh = row[0] << -u;
        } else {
            const int w = u / 32, shift = u % 32;
            fresh = __funnelshift_r(row[w], w + 1 < a.words ? row[w + 1] : 0u, shift);
        }
        bits |= fresh & low_bits(it.count - u) & ~low_bits(-u);
    }
    return bits;
}

__device__ __forceinline__ bool has_page(const PagedAttention& a, int b, int slot) {
    const int page = a.table[static_cast<int64_t>(b) * a.table_stride + (slot >> a.page_shift)];
    return page >= 0 && page < a.pages;
}

// Waits for phase `parity` of `bar`; false after some seconds.
__device__ __forceinline__ bool wait_counted(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
        "mov.u32 n, 0;\n\t"
        "TRY:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@p bra DONE;\n\t"
        "add.u32 n, n, 1;\n\t"
        "setp.lt.u32 q, n, 33554432;\n\t"
        "@q bra TRY;\n\t"
        "DONE:\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16-bit types: pairs, exponents.
template <typename T>
struct Half16;
template <>
struct Half16<__half> {
    static constexpr uint32_t kExponent = 0x7c007c00u;
    static constexpr uint32_t kUmma = 0;  // the operands' type in tcgen05.mma's descriptor
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct Half16<__nv_bfloat16> {
    static constexpr uint32_t kExponent = 0x7f807f80u;
    static constexpr uint32_t kUmma = 1u << 7 | 1u << 10;
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
// Bits 15 and 31 where one of a word's two values is an infinity or NaN: a carry out of the
// exponent.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return ((w & 0x7fff7fffu) + (0x80008000u - Half16<T>::kExponent)) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {  // 0 in place of such values
    return w & ~((not_finite<T>(w) >> 15) * 0xffffu);
}
// A result that an infinite value has reached is NaN like one that a NaN has.
__device__ __forceinline__ float nan_if_infinite(float y) { return fmaf(y, 0.0f, y); }

// Four dims of a result, `at` elements into out (a multiple of 4).
template <typename T>
__device__ __forceinline__ void put4(const PagedAttention& a, int64_t at, float4 y) {
    if (a.out_f32) {
        float* const to = static_cast<float*>(a.out) + at;
        if (a.aligned & 2) *reinterpret_cast<float4*>(to) = y;
        else to[0] = y.x, to[1] = y.y, to[2] = y.z, to[3] = y.w;
    } else {
        const uint2 w = make_uint2(Half16<T>::pack(y.x, y.y), Half16<T>::pack(y.z, y.w));
        uint16_t* const to = static_cast<uint16_t*>(a.out) + at;
        if (a.aligned & 2) *reinterpret_cast<uint2*>(to) = w;
        else to[0] = w.x & 0xffffu, to[1] = w.x >> 16, to[2] = w.y & 0xffffu, to[3] = w.y >> 16;
    }
}
}  // namespace paged
#endif

}  // namespace kt
