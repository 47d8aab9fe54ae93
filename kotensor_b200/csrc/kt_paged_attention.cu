// kt_paged_attention.cu -- attention over the paged 16-bit key/value cache, for few query
// vectors a key/value head (single tokens), and the choice of the kernel.
//
// Row t of sequence b with n = lengths[b]: for each query head, over the slots j it sees
// (all j < n, and of this call's tokens those that its mask or the order of rows allows),
//   s_j = scale * (q . K_j),  out = sum_j softmax(s)_j V_j,   0 where it sees nothing.
//
// Sixteen query vectors that share a key/value head (rows x heads of a group) are an item,
// over tiles of 128 slots.  A warp has 16 slots of each tile, which one m16n8k16 product
// after the other takes as they lie: keys as the first product's B, values, transposed by
// the load, as the second's; scores leave the first in the layout in which the second reads
// probabilities.  Every warp keeps its own largest scores and sums, in fp32; an item's end
// brings them together.  Probabilities are rounded to the cache's type, half a step of each
// (2^-8 of it in bfloat16, 2^-11 in fp16) as a 16-bit result itself is at the end; they are
// all of an fp32 result's error, 8e-4 of its size in bfloat16.  The products take no wider ones,
// and two terms each would double the second product.
//
// A ninth warp copies: the pages of a tile as swizzled boxes of 64 dims by TMA, keys and
// values in turn through a ring of 160 KB, so that some 100 KB are on their way to an SM at
// any time and across the ends of items.  (Two CTAs of four warps with rings of 80 KB: 231 us
// where this takes 224, and 37 parts to merge where this leaves 18, 93 where this takes 84.)
// Bound by memory: 64 sequences of 3001 to 8190 tokens, 8 heads of 128, 222 to 225 us, 6.5 to 6.6
// TB/s; one of 120001 82 to 84 us, 5.9 TB/s, of which about 5 go into the merge.  By latency when short: 301
// tokens 7.4 us, of which a tile's chain of copy, product, exponentials and product is 1.5.
#include <algorithm>

#include "kt_paged.h"

namespace kt {
namespace {

using namespace paged;

constexpr int kWarps = 8;                        // that compute; one more copies
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kVectors = 16;                     // query vectors of an item (the product's M)
constexpr int kTile = 128;                       // slots of a tile, 16 to a warp
// What entering an item costs, in tiles (8 sequences of 5000 tokens, 8 heads of 128: 33.2 us, counted as two tiles
// 34.6), and up to how many an item is not cut (300 tokens 8.2 us, cut into single tiles 9.7; 1000 tokens cut so
// 9.6, into fours 13.5).
constexpr int kStart = 4, kLeast = 1, kWhole = 3;
// Probabilities are kept 2^kLift times larger: in fp16 those down to 2^-36 of the largest
// stay clear of underflow; the factor cancels in the division by their sum.
constexpr float kLift = 12.0f;

template <int HDP>
struct RowsShape {
    static constexpr int kBlocks = HDP / 64;               // blocks of 64 dims: swizzled rows of 128 bytes
    static constexpr int kUnit = kBlocks * kTile * 128;    // the keys or the values of a tile
    static constexpr int kUnits = 160 * 1024 / kUnit;      // in the ring: keys, values, keys, ...
    static constexpr int kPitch = HDP + 4;
    static constexpr int kArea = kUnits * kUnit;           // sums of four pairs of warps; the queries before
    static constexpr int kQPitch = HDP * 2 + 16;
    static constexpr int kStats = kArea + 4 * kVectors * kPitch * 4;  // largest score, sum of each warp's vectors
    static constexpr int kTotals = kStats + 2 * kWarps * kVectors * 4;
    static constexpr int kBars = kTotals + 2 * kVectors * 4;
    static constexpr int kValid = kBars + 16 * kUnits;     // boxes of a unit that have a page
    static constexpr int kSmem = 1024 + kValid + 4 * kUnits;
    static constexpr int kPart = kVectors * (HDP + 2);     // floats of a part: sums, largest scores, totals
    static_assert(kSmem <= 232448 && kVectors * kQPitch <= kStats - kArea, "shared memory");
};

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void matrices(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void matrices_turned(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Sums over the parts' own references -> the common one's (0 where nothing was summed).
__device__ __forceinline__ float weigh(float reference, float sum, float common) {
    return sum == 0.0f ? 0.0f : ex2(reference - common);
}

template <typename T, int HDP>
__global__ void __launch_bounds__(kThreads, 1) paged_rows_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                 const __grid_constant__ CUtensorMap v_map,
                                                                 const __grid_constant__ PagedAttention a,
                                                                 int32_t* __restrict__ err) {
    using S = RowsShape<HDP>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ int last_cta;
    const uint32_t raw = dev::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* const smem = smem_raw + (base - raw);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, d = a.head_dim;
    auto full = [&](int x) { return base + S::kBars + 16 * x; };
    auto empty = [&](int x) { return base + S::kBars + 16 * x + 8; };
    volatile uint32_t* const with_page = reinterpret_cast<uint32_t*>(smem + S::kValid);
    if (threadIdx.x == 0) {
        for (int x = 0; x < S::kUnits; ++x) {
            dev::mbar_init(full(x), 1);
            dev::mbar_init(empty(x), kWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 32) {
        dev::prefetch_map(&k_map);
        dev::prefetch_map(&v_map);
    }
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    __shared__ Plan<kWarps + 1> plan;
    const WorkList<kWarps + 1, kVectors, kTile, kStart, kLeast, kWhole, 0> work{a, plan};
    if (!work.start()) {  // (its barriers also publish the mbarriers)
        if (warp == kWarps) zero_rows(a);
        return;
    }
    const Item& it = plan.at[warp];
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {  // a lane that has given up goes on without waiting
        if (ok && !wait_counted(bar, parity)) ok = false;
    };

    if (warp == kWarps) {
        // Copies: a lane has a box (64 dims of the slots of a page, at most a tile's) of the keys' or values' unit.
        const int box = min(kPagedBox, 1 << a.page_shift), boxes = kTile / box;  // 16, 32 or 64 slots; 8, 4 or 2 to a tile
        const int mine = lane % boxes, block = lane / boxes % S::kBlocks;
        const bool copies = lane < boxes * S::kBlocks;
        Ring<S::kUnits> ring;
        int units = 0;  // at most kUnits: those that may be in flight
        do {
            for (int tile = it.from, to = it.to; tile < to; ++tile) {
                const int slot = tile * kTile + mine * box;
                int page = -1;
                if (copies && slot < it.sees) page = a.table[static_cast<int64_t>(it.b) * a.table_stride + (slot >> a.page_shift)];
                const bool here = page >= 0 && page < a.pages;
                const uint32_t who = __ballot_sync(0xffffffffu, here);
                const int row = here ? ((page * a.kv_heads + it.head) << a.page_shift) + (slot & ((1 << a.page_shift) - 1)) : 0;
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int x = ring.at;
                    if (units == S::kUnits) wait(empty(x), ring.phase ^ 1);
                    if (!__all_sync(0xffffffffu, ok)) break;
                    units = min(units + 1, S::kUnits);
                    ring.next();
                    if (lane == 0) {
                        with_page[x] = who & ((1u << boxes) - 1u);
                        dev::mbar_expect_tx(full(x), __popc(who) * box * 128);
                    }
                    __syncwarp();
                    if (here)
                        dev::tma_load_2d(base + x * S::kUnit + block * (kTile * 128) + mine * box * 128, v ? &v_map : &k_map,
                                         block * 64, row, full(x));
                }
                if (!__all_sync(0xffffffffu, ok)) break;
            }
        } while (__all_sync(0xffffffffu, ok) && work.next());
        zero_rows(a);
        // no copy is in flight past this point, also where a wait has given up
        if (units == S::kUnits) ring.phase ^= 1;  // the oldest one is at the ring's place, of the round before
        else ring.at = 0;
        for (; units > 0; --units, ring.next())
            if (!wait_counted(full(ring.at), ring.phase)) ok = false;
        if (!ok) atomicOr(err, 1);
        return;
    }

    const int r8 = lane / 4, t4 = lane % 4;
    float* const area = reinterpret_cast<float*>(smem + S::kArea);
    float* const stats = reinterpret_cast<float*>(smem + S::kStats);    // [warp][vector]: largest scores, then sums
    float* const totals = reinterpret_cast<float*>(smem + S::kTotals);  // [vector]
    float* const parts = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + kPagedPartsAt);
    Ring<S::kUnits> ring;
    do {
        const int from = it.from, to = it.to;
        if (from >= to) continue;
        // the item's queries, through shared memory; this thread's vectors are r8 and r8 + 8
        {
            constexpr int kPieces = HDP / 8;
            const int vec = threadIdx.x / kPieces, dim = threadIdx.x % kPieces * 8;
            if (vec < kVectors) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (vec < it.valid && dim < d) {
                    const uint16_t* const from_q = static_cast<const uint16_t*>(a.q) + place_of(a, it.b, it.head, it.v0 + vec, a.q_stride) + dim;
                    if (a.aligned & 1) {
                        w = *reinterpret_cast<const uint4*>(from_q);
                    } else {
                        uint32_t e[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) e[j] = from_q[2 * j] | static_cast<uint32_t>(from_q[2 * j + 1]) << 16;
                        w = make_uint4(e[0], e[1], e[2], e[3]);
                    }
                }
                *reinterpret_cast<uint4*>(smem + S::kArea + vec * S::kQPitch + dim * 2) = w;
            }
        }
        const int t[2] = {r8 < it.valid ? (it.v0 + r8) / a.group : -1, r8 + 8 < it.valid ? (it.v0 + r8 + 8) / a.group : -1};
        compute_sync();
        uint32_t q[HDP / 16][4];
#pragma unroll
        for (int s = 0; s < HDP / 16; ++s)
            matrices(base + S::kArea + (lane % 16) * S::kQPitch + (16 * s + lane / 16 * 8) * 2, q[s]);
        // slots that all of the item's vectors see
        const int clear = a.visible ? it.held : min(it.held + it.v0 / a.group + 1, it.sees);
        float o[HDP / 8][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < HDP / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        for (int tile = from; tile < to; ++tile) {
            const int kx = ring.at;
            const uint32_t k_phase = ring.phase;
            ring.next();
            const int vx = ring.at;
            const uint32_t v_phase = ring.phase;
            ring.next();
            const int slot = tile * kTile + warp * 16;
            float s[2][4] = {};
            wait(full(kx), k_phase);
            __syncwarp();
            if (slot < it.sees) {
                const uint32_t k_row = base + kx * S::kUnit + (warp * 16 + lane % 8 + lane / 16 * 8) * 128;
#pragma unroll
                for (int i = 0; i < HDP / 16; ++i) {
                    uint32_t m[4];
                    matrices(k_row + i / 4 * (kTile * 128) + (((2 * (i % 4) + lane / 8 % 2) ^ (lane % 8)) << 4), m);
                    mma<T>(s[0], q[i], m[0], m[1]);
                    mma<T>(s[1], q[i], m[2], m[3]);
                }
            }
            const uint32_t pages = with_page[kx];
            __syncwarp();
            if (lane == 0) dev::mbar_arrive(empty(kx));
            uint32_t p[4] = {0, 0, 0, 0};
            const bool page = pages >> (warp * 16 / min(kPagedBox, 1 << a.page_shift)) & 1u;
            const bool edge = slot + 16 > clear || !page;
            uint32_t seen[2] = {0xffffu, 0xffffu};
            if (edge) {
#pragma unroll
                for (int i = 0; i < 2; ++i) seen[i] = t[i] >= 0 && page ? seen_bits(a, it, t[i], slot) & 0xffffu : 0u;
            }
            if (slot < it.sees) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float z[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {  // slots 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9
                        z[e] = s[e / 2][2 * i + e % 2] * a.factor;
                        if (edge && !(seen[i] >> (2 * t4 + e % 2 + e / 2 * 8) & 1u)) z[e] = -INFINITY;
                    }
                    float high = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 1));
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 2));
                    const float now = fmaxf(top[i], high), less = now == -INFINITY ? 0.0f : now - kLift;
                    const float fade = top[i] == -INFINITY ? 0.0f : ex2(top[i] - now);
                    top[i] = now;
                    if (__any_sync(0xffffffffu, fade != 1.0f)) {
                        sum[i] = sum[i] == 0.0f ? 0.0f : sum[i] * fade;
#pragma unroll
                        for (int j = 0; j < HDP / 8; ++j) o[j][2 * i] *= fade, o[j][2 * i + 1] *= fade;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        z[e] = ex2(z[e] - less);
                        sum[i] += z[e];
                    }
                    p[i] = Half16<T>::pack(z[0], z[1]);
                    p[i + 2] = Half16<T>::pack(z[2], z[3]);
                }
            }
            wait(full(vx), v_phase);
            __syncwarp();
            if (edge && slot < it.sees) {
                // What no vector sees counts nothing, whatever it is: its rows of the tile become zeros.  A value that is
                // not finite counts for those that see it alone, who get NaN in its dim; a zero takes its place.
                const uint32_t any = __reduce_or_sync(0xffffffffu, seen[0] | seen[1]);
                const int row = lane / 2;
                unsigned char* const rows = smem + vx * S::kUnit + warp * 16 * 128;
                uint4* const line = reinterpret_cast<uint4*>(rows + row * 128);
                uint32_t over = 0;
#pragma unroll
                for (int i = 0; i < HDP / 16; ++i) {
                    const int piece = lane % 2 * (HDP / 16) + i;
                    const uint4 w = line[piece / 8 * (kTile * 128 / 16) + piece % 8];
                    over |= not_finite<T>(w.x) | not_finite<T>(w.y) | not_finite<T>(w.z) | not_finite<T>(w.w);
                }
                const bool hidden = !(any >> row & 1u);
                for (uint32_t told = __ballot_sync(0xffffffffu, over != 0 && !hidden); told != 0;) {
                    const int r = (__ffs(told) - 1) / 2;
                    told &= ~(3u << (2 * r));
#pragma unroll
                    for (int j = 0; j < HDP / 8; ++j) {
                        const uint32_t bad = not_finite<T>(
                            *reinterpret_cast<const uint32_t*>(rows + j / 8 * (kTile * 128) + r * 128 + ((j % 8 ^ (r & 7)) << 4) + 4 * t4));
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if ((e % 2 ? bad >> 31 : bad & 0x8000u) && (seen[e / 2] >> r & 1u)) o[j][e] = __uint_as_float(0x7fc00000u);
                    }
                }
                __syncwarp();
                if (hidden) {
#pragma unroll
                    for (int i = 0; i < HDP / 16; ++i) {
                        const int piece = lane % 2 * (HDP / 16) + i;
                        line[piece / 8 * (kTile * 128 / 16) + piece % 8] = make_uint4(0, 0, 0, 0);
                    }
                } else if (over != 0) [[unlikely]] {
#pragma unroll 1
                    for (int i = 0; i < HDP / 16; ++i) {
                        const int piece = lane % 2 * (HDP / 16) + i;
                        uint4& w = line[piece / 8 * (kTile * 128 / 16) + piece % 8];
                        w = make_uint4(finite_part<T>(w.x), finite_part<T>(w.y), finite_part<T>(w.z), finite_part<T>(w.w));
                    }
                }
                __syncwarp();
            }
            if (slot < it.sees) {
                const uint32_t v_row = base + vx * S::kUnit + (warp * 16 + lane % 16) * 128;
#pragma unroll
                for (int j = 0; j < HDP / 16; ++j) {
                    uint32_t m[4];
                    matrices_turned(v_row + j / 4 * (kTile * 128) + (((2 * (j % 4) + lane / 16) ^ (lane % 8)) << 4), m);
                    mma<T>(o[2 * j], p, m[0], m[1]);
                    mma<T>(o[2 * j + 1], p, m[2], m[3]);
                }
            }
            if (edge) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy to these rows
            __syncwarp();
            if (lane == 0) dev::mbar_arrive(empty(vx));
        }
        // the warps' sums, brought to a common reference and added in a fixed order
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
            if (t4 == 0) {
                stats[warp * kVectors + r8 + 8 * i] = top[i];
                stats[(kWarps + warp) * kVectors + r8 + 8 * i] = sum[i];
            }
        }
        compute_sync();
        float common[2], by[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int v = r8 + 8 * i;
            common[i] = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) common[i] = fmaxf(common[i], stats[w * kVectors + v]);
            by[i] = weigh(top[i], sum[i], common[i]);
            if (warp == 0 && t4 == 0) {
                float total = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float m = stats[w * kVectors + v], l = stats[(kWarps + w) * kVectors + v];
                    total += weigh(m, l, common[i]) * l;
                }
                totals[v] = common[i], totals[kVectors + v] = total;
            }
        }
        float* const sums = area + (warp % 4) * (kVectors * S::kPitch);
#pragma unroll
        for (int step = 0; step < 2; ++step) {
            if (warp / 4 == 1 - step) {
#pragma unroll
                for (int j = 0; j < HDP / 8; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float2* const at = reinterpret_cast<float2*>(sums + (r8 + 8 * i) * S::kPitch + 8 * j + 2 * t4);
                        const float2 f = step == 0 ? make_float2(0.0f, 0.0f) : *at;
                        *at = make_float2(f.x + o[j][2 * i] * by[i], f.y + o[j][2 * i + 1] * by[i]);
                    }
            }
            compute_sync();
        }
        // dims dim .. dim + 3 of vector `vec`, from their sums and the vector's total
        auto finish = [&](int vec, int dim, float4 y, float total) {
            if (dim >= d) return;
            const int64_t at = place_of(a, it.b, it.head, it.v0 + vec, static_cast<int64_t>(a.heads) * d) + dim;
            const float scale = total == 0.0f ? 0.0f : 1.0f / total;
            put4<T>(a, at, make_float4(nan_if_infinite(y.x * scale), nan_if_infinite(y.y * scale), nan_if_infinite(y.z * scale), nan_if_infinite(y.w * scale)));
        };
        const bool whole = from == 0 && to == it.tiles;
        // the part of an item that an earlier CTA began is the CTA's part 0, of one that goes on its part 1
        float* const part = parts + (static_cast<int64_t>(blockIdx.x) * 2 + (from == 0)) * S::kPart;
        for (int e = threadIdx.x; e < it.valid * (HDP / 4); e += kWarps * 32) {
            const int vec = e / (HDP / 4), dim = e % (HDP / 4) * 4;
            float4 y = *reinterpret_cast<const float4*>(area + vec * S::kPitch + dim);
#pragma unroll
            for (int i = 1; i < 4; ++i) {
                const float4 z = *reinterpret_cast<const float4*>(area + (i * kVectors + vec) * S::kPitch + dim);
                y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
            }
            if (whole) finish(vec, dim, y, totals[kVectors + vec]);
            else __stcg(reinterpret_cast<float4*>(part + vec * HDP + dim), y);
        }
        if (!whole) {
            if (threadIdx.x < 2 * kVectors) __stcg(part + kVectors * HDP + threadIdx.x, totals[threadIdx.x]);
            const int c0 = work.first_cta(it), c1 = work.last_cta(it);
            int32_t* const counter = static_cast<int32_t*>(a.scratch) + c0;
            __threadfence();
            compute_sync();
            if (threadIdx.x == 0) last_cta = dev::atomic_add_acq_rel(counter, 1) == c1 - c0;
            compute_sync();
            if (last_cta) {
                __threadfence();
                const int n = c1 - c0 + 1;
                const float* const from_c0 = parts + static_cast<int64_t>(c0) * 2 * S::kPart;
                for (int e = threadIdx.x; e < it.valid * (HDP / 4); e += kWarps * 32) {
                    const int vec = e / (HDP / 4), dim = e % (HDP / 4) * 4;
                    float top = -INFINITY, total = 0.0f;
                    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    constexpr int kBatch = 8;  // parts whose loads are under way together (one by one 37 took 20 us)
                    for (int i = 0; i < n; i += kBatch) {
                        float ref[kBatch], sum[kBatch];
                        float4 f[kBatch];
#pragma unroll
                        for (int j = 0; j < kBatch; ++j) {
                            // the first is its CTA's part 1, the others are their CTAs' parts 0
                            const float* const p = from_c0 + static_cast<int64_t>(i + j == 0 ? 1 : 2 * min(i + j, n - 1)) * S::kPart;
                            ref[j] = __ldcg(p + kVectors * HDP + vec);
                            sum[j] = __ldcg(p + kVectors * (HDP + 1) + vec);
                            f[j] = __ldcg(reinterpret_cast<const float4*>(p + vec * HDP + dim));
                        }
                        float now = top;
#pragma unroll
                        for (int j = 0; j < kBatch; ++j) now = fmaxf(now, ref[j]);
                        const float fade = total == 0.0f ? 0.0f : ex2(top - now);
                        top = now;
                        total *= fade, y.x *= fade, y.y *= fade, y.z *= fade, y.w *= fade;
#pragma unroll
                        for (int j = 0; j < kBatch; ++j) {
                            const float l = i + j < n ? sum[j] : 0.0f, w = weigh(ref[j], l, top);
                            total += w * l;
                            y.x = fmaf(w, f[j].x, y.x), y.y = fmaf(w, f[j].y, y.y), y.z = fmaf(w, f[j].z, y.z), y.w = fmaf(w, f[j].w, y.w);
                        }
                    }
                    finish(vec, dim, y, total);
                }
                if (threadIdx.x == 0) *counter = 0;
            }
        }
        compute_sync();  // the areas and last_cta are free again
    } while (work.next());
    if (!ok) atomicOr(err, 1);
}

template <typename T, int HDP>
cudaError_t launch_rows(const CUtensorMap& k_map, const CUtensorMap& v_map, const PagedAttention& a, int sm_count,
                        int32_t* err, cudaStream_t s) {
    using S = RowsShape<HDP>;
    static std::atomic<uint64_t> allowed{0};
    const auto kernel = paged_rows_kernel<T, HDP>;
    cudaError_t e = allow_shared(kernel, S::kSmem, allowed);
    if (e != cudaSuccess) return e;
    const int64_t items = static_cast<int64_t>(a.batch) * a.kv_heads * ((static_cast<int64_t>(a.rows) * a.group + kVectors - 1) / kVectors);
    const int64_t most = std::max(items, items * ((a.capacity + kTile - 1) / kTile) / kLeast);
    const int grid = static_cast<int>(std::min<int64_t>(std::min(sm_count, kPagedRowsCtas), most));
    return launch_dependent(kernel, dim3(grid), dim3(kThreads), S::kSmem, s, k_map, v_map, a, err);
}

}  // namespace

size_t paged_rows_bytes() { return static_cast<size_t>(kPagedRowsCtas) * 2 * RowsShape<128>::kPart * sizeof(float); }

cudaError_t launch_paged_attention(const Paged& c, int layer, const PagedAttention& a, int sm_count, int32_t* err,
                                   cudaStream_t s) {
    const int64_t rows = static_cast<int64_t>(c.pages) * c.kv_heads * c.page, row_bytes = 2ll * c.head_dim;
    CUtensorMap maps[2];
    for (int v = 0; v < 2; ++v)
        if (!encode_tmap_2d(&maps[v], c.dtype == KT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                            static_cast<const char*>(v ? c.values : c.keys) + layer * rows * row_bytes, c.head_dim, rows, row_bytes,
                            64, std::min(c.page, kPagedBox), CU_TENSOR_MAP_SWIZZLE_128B))
            return cudaErrorInvalidValue;
    // Which kernel is the faster.  This file's reads the cache once for every sixteen vectors, the other one once for
    // 256, but takes 4 us longer to enter, leave and merge.  So this one runs for sixteen vectors or fewer; for up to 32
    // while its items leave no SM two (20 vectors of 32 heads over 8 of 128, 1 / 8 / 64 sequences of 300 tokens: 9.2 /
    // 9.4 / 57 us here, 14.7 / 17.6 / 57 there; 8 sequences of 4000: 43, 56); and for more where they are very few (112
    // vectors of 14 heads over 2 of 64, 1 / 8 sequences: 300 tokens 7.6 / 8.6 us here, 12.6 / 12.6 there, 20000 and 4000 tokens
    // 22 / 33 here, 27 / 17 there).  Sequences past some 20000 slots are not told apart, which costs the most vectors that
    // stay here: 100000 slots of one head of 128, 64 / 128 / 256 vectors 41 / 61 / 104 us here, 53 / 55 / 55 there (20000 slots
    // 21 / 23 / 31 and 28 / 30 / 31); of two of 64, 56 / 112 vectors 46 / 72 us here, 36 / 37 there.
    const int64_t sixteens = (static_cast<int64_t>(a.rows) * a.group + kVectors - 1) / kVectors, items = sixteens * a.batch * a.kv_heads;
    if (sixteens > 1 && items > (sixteens == 2 ? sm_count : 16)) return launch_paged_many(c.dtype == KT_BF16, maps, a, sm_count, err, s);
    const bool bf16 = c.dtype == KT_BF16, wide = c.head_dim > 64;
    const auto launch = bf16 ? wide ? launch_rows<__nv_bfloat16, 128> : launch_rows<__nv_bfloat16, 64>
                             : wide ? launch_rows<__half, 128> : launch_rows<__half, 64>;
    return launch(maps[0], maps[1], a, sm_count, err, s);
}

}  // namespace kt
