// kt_kv8_prompt.cu -- attention of many query rows over the 8-bit key/value cache
// (a prompt, or a chunk of one) on the 5th-generation tensor cores.
//
// A CTA owns 128 query vectors that share a key/value head: rows x heads of the
// group, in row order.  Over tiles of 128 slots,
//   S = Q K^T,   P = 2^(S * scale - reference) * value scale,   O += P V,
// with the codes of K and V exact in fp16 and Q and P as two fp16 terms each
// (kt_kv8_attention.cu), so each product is two tcgen05.mma chains into one fp32
// accumulator: 4 x 128 x 128 x head_dim x 2 operations a tile.
//
// Even tiles and odd tiles are two streams with their own S, O, running maximum and
// sum: while four warps turn one stream's S into P, the tensor cores work on the
// other's products.  They meet once, at the end.  Tensor memory: S of stream x in
// columns 128 x .., where P replaces it (a thread owns one vector, lane and row of
// both: 32 scores read, 16 + 16 columns of hi and lo pairs written back in their
// place); O of stream x in columns 256 + HDP x ...
//   warps 0-3, 4-7  softmax of stream 0, 1, and their share of the epilogue
//   warps 8-11      codes -> fp16, K and V tiles in 128-byte swizzled rows of 64 dims
//                   (K-major for the first product, MN-major for the second: the
//                   same bytes, another descriptor)
//   warp 12         issues the products
//
// References.  The sum l is relative to the running maximum D of the scores.  The
// numerators carry the values' scales, which may differ by any factor from block
// to block, so they are relative to a reference R of their own, the maximum of
// score + log2(value scale): both terms of P keep 22 bits of what matters to O.
// R moves only when the maximum passes it by 2^kSlack, so O is seldom rescaled.
#include <cuda_fp16.h>

#include "kt_kv8.h"

namespace kt {
namespace {

constexpr int kVecTile = 128;   // query vectors of a CTA (the MMA's M)
constexpr int kSlots = 128;     // slots of a tile (the first product's N, the second's K)
constexpr int kSoftmaxWarps = 8;
constexpr int kConvertWarps = 4;
constexpr int kMmaWarp = kSoftmaxWarps + kConvertWarps;
constexpr int kThreads = (kMmaWarp + 1) * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLift = 7.0f;   // numerators are 2^kLift larger, up to 2^(kLift + kSlack) <= 2^15
constexpr float kSlack = 8.0f;

template <int HDP>
struct PromptShape {
    static constexpr int kBlocks = HDP / 64;              // blocks of 64 dims: 128-byte rows
    static constexpr int kTile = kBlocks * kSlots * 128;  // fp16 tile of 128 rows
    static constexpr int kQ = 0, kK = 2 * kTile, kV = 4 * kTile, kEnd = 6 * kTile;
    static constexpr int kOutPitch = kVecTile + 1;        // epilogue: [dim][vector], over K and V
    static constexpr int kSmem = 1024 + kEnd + kVecTile * 4 + 256;
    static_assert(HDP * kOutPitch * 4 + 3 * kVecTile * 4 <= 4 * kTile + 4096, "epilogue area");
    static_assert(kSmem <= 232448, "shared memory per CTA");
};

__device__ __forceinline__ uint64_t desc_base(uint32_t addr, uint32_t lead) {
    // 128-byte swizzle, atoms of 8 rows 1024 bytes apart, descriptor version 1
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
           (static_cast<uint64_t>(2) << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Waits for the loads in flight; r, read by one of them, passes through so that no
// use of it can move ahead of the wait.
__device__ __forceinline__ void wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 columns of this warp's 32 lanes, in flight until wait_ld.
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ void two_terms(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(x0 - f.x, x1 - f.y));
}
// Two of four codes as fp16: flipped sign bits, 0x64xx = 1024 + xx, less 1152.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t flipped) {
    const uint32_t r = dev::prmt(flipped, 0x64646464u, kSel);
    return h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&r), __half2half2(__ushort_as_half(0x6480))));
}
// Byte offset of 16-byte piece `piece` (of 64 dims: 8) of row `row` in a swizzled block.
__device__ __forceinline__ uint32_t swizzled(int row, int piece) {
    return static_cast<uint32_t>(row * 128 + ((piece ^ (row & 7)) << 4));
}

template <int HDP>
__global__ void __launch_bounds__(kThreads, 1) kv8_prompt_kernel(Kv8Attention a, int aligned, float* __restrict__ lse,
                                                                 int32_t* __restrict__ err) {
    using S = PromptShape<HDP>;
    dev::pdl_wait();
    const Kv8& c = a.cache;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, d = c.head_dim;
    const int b = blockIdx.z, h = blockIdx.y;
    const int vt = gridDim.x - 1 - blockIdx.x;  // the rows that see most first
    const int group = a.heads / c.kv_heads, vectors = a.rows_per_seq * group, v0 = vt * kVecTile;
    const int rows = kv8_rows(a.counts, b, a.rows_per_seq), held = kv8_held(c, b);
    const int seen = min(held + rows, c.capacity);
    const int64_t head = static_cast<int64_t>(b) * c.kv_heads + h;
    // where vector v's query and output lie
    auto place = [&](int v, int64_t stride) {
        return (static_cast<int64_t>(b) * a.rows_per_seq + v / group) * stride + static_cast<int64_t>(h * group + v % group) * d;
    };
    // rows that are no tokens
    for (int v = max(v0, rows * group) + warp; v < min(v0 + kVecTile, vectors); v += kThreads / 32)
        for (int i = lane; i < d; i += 32) a.context[place(v, static_cast<int64_t>(a.heads) * d) + i] = 0.0f;
    const int real = min(kVecTile, rows * group - v0);  // vectors of this tile that are
    if (real <= 0) {
        dev::pdl_launch_dependents();
        return;
    }
    const int most = min(held + (v0 + real - 1) / group + 1, seen);  // slots its last vector sees
    const int tiles = (most + kSlots - 1) / kSlots;

    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = dev::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* const smem = smem_raw + (base - raw);
    float* const q_factor = reinterpret_cast<float*>(smem + S::kEnd);
    const uint32_t bars = base + S::kEnd + kVecTile * 4;
    auto k_full = [&](int x) { return bars + 8 * x; };
    auto k_free = [&](int x) { return bars + 16 + 8 * x; };
    auto v_full = [&](int x) { return bars + 32 + 8 * x; };
    auto v_free = [&](int x) { return bars + 48 + 8 * x; };
    auto s_full = [&](int x) { return bars + 64 + 8 * x; };
    auto p_full = [&](int x) { return bars + 80 + 8 * x; };
    const uint32_t done = bars + 96;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kEnd + kVecTile * 4 + 104);
    if (threadIdx.x == 0) {
        for (int x = 0; x < 2; ++x) {
            dev::mbar_init(k_full(x), kConvertWarps);
            dev::mbar_init(k_free(x), 1);
            dev::mbar_init(v_full(x), kConvertWarps);
            dev::mbar_init(v_free(x), 1);
            dev::mbar_init(s_full(x), 1);
            dev::mbar_init(p_full(x), 4);
        }
        dev::mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dev::smem_u32(tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *tmem_slot;
    // only now: a dependent kernel's CTA on this SM must not take the tensor memory first
    dev::pdl_launch_dependents();

    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {  // one lane
        if (!dev::mbar_wait_bounded(bar, parity)) {
            ok = false;
            atomicOr(err, 1);
        }
        return ok;
    };
    auto wait_all = [&](uint32_t bar, uint32_t parity) {  // a warp: its lanes go on, or give up, together
        return __all_sync(0xffffffffu, wait(bar, parity));
    };
    // The state of a softmax thread: vector v0 + row of stream x.
    const int x = warp / 4, row = (warp % 4) * 32 + lane;
    float D = -INFINITY, R = -INFINITY, l = 0.0f;

    if (warp < kSoftmaxWarps) {
        // Queries, a warp to a vector, a lane to four dims: scaled by a power of two to
        // at most 1 and split into two terms; a negative scale turns the query's sign.
        for (int v = warp; v < kVecTile; v += kSoftmaxWarps) {
            float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const int dim = 4 * lane;
            if (v < real && dim < d) {
                const float* q = a.q + place(v0 + v, a.q_stride) + dim;
                if (aligned & 1) {
                    const float4 t = *reinterpret_cast<const float4*>(q);
                    f[0] = t.x, f[1] = t.y, f[2] = t.z, f[3] = t.w;
                } else {
                    f[0] = q[0], f[1] = q[1], f[2] = q[2], f[3] = q[3];
                }
            }
            uint32_t top = 0;  // the largest exponent, by the bits of |q|; NaN counts as infinity
            for (int i = 0; i < 4; ++i) top = max(top, min(__float_as_uint(f[i]) & 0x7fffffffu, 0x7f800000u));
            top = __reduce_max_sync(0xffffffffu, top);
            const int e = min(max(static_cast<int>(top >> 23) - 126, -126), 126);
            float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            if (a.scale < 0.0f) down = -down;
            if (lane == 0) q_factor[v] = fabsf(a.scale) * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            if (dim < HDP) {
                uint2 hi, lo;
                two_terms(f[0] * down, f[1] * down, hi.x, lo.x);
                two_terms(f[2] * down, f[3] * down, hi.y, lo.y);
                const uint32_t at = S::kQ + (dim / 64) * (kVecTile * 128) + swizzled(v, dim % 64 / 8) + (lane & 1) * 8;
                *reinterpret_cast<uint2*>(smem + at) = hi;
                *reinterpret_cast<uint2*>(smem + at + S::kTile) = lo;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("bar.sync 1, %0;" ::"n"((kSoftmaxWarps + 1) * 32) : "memory");

        const uint32_t s_tm = tmem + (static_cast<uint32_t>(row & ~31) << 16) + x * kSlots;
        const uint32_t o_tm = tmem + (static_cast<uint32_t>(row & ~31) << 16) + 2 * kSlots + x * HDP;
        const float factor = q_factor[row];
        const int limit = row < real ? min(held + (v0 + row) / group + 1, seen) : 0;
        const float* k_scales = c.k_scales + head * (c.capacity / c.block);
        const float* v_scales = c.v_scales + head * (c.capacity / c.block);
        for (int i = x, it = 0; i < tiles; i += 2, ++it) {
            const int first = i * kSlots;
            float ks[8], vs[8];
#pragma unroll
            for (int g = 0; g < 8; ++g) {  // a block the vector does not see has no scale, whatever is there
                const bool in = first + 16 * g < limit;
                const int at = in ? (first + 16 * g) / c.block : 0;
                ks[g] = in ? k_scales[at] * factor : 0.0f;
                vs[g] = in ? v_scales[at] : 0.0f;
            }
            if (!wait_all(s_full(x), it & 1)) break;
            tc_after();
            const bool edge = __any_sync(0xffffffffu, first + kSlots > limit);
            // the largest score of each 16 slots
            float top[8];
            uint32_t s[2][32];
            ld32(s_tm, s[0]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                wait_ld(s[q & 1]);
                if (q < 3) ld32(s_tm + 32 * (q + 1), s[(q + 1) & 1]);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    float m = -INFINITY;
                    if (edge) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (first + 32 * q + 16 * g + j < limit) m = fmaxf(m, __uint_as_float(s[q & 1][16 * g + j]));
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) m = fmaxf(m, __uint_as_float(s[q & 1][16 * g + j]));
                    }
                    top[2 * q + g] = m == -INFINITY ? m : m * ks[2 * q + g];
                }
            }
            ld32(s_tm, s[0]);
            float new_d = D, most_w = -INFINITY;
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                new_d = fmaxf(new_d, top[g]);
                most_w = fmaxf(most_w, top[g] + __log2f(vs[g]));
            }
            const float ref = new_d == -INFINITY ? 0.0f : new_d;
            l = D == -INFINITY ? l : l * ex2(D - ref);
            D = new_d;
            const bool move = most_w > R + kSlack || (R == -INFINITY && most_w > R);
            if (__any_sync(0xffffffffu, move)) {
                const float fade = !move ? 1.0f : R == -INFINITY ? 0.0f : ex2(R - most_w);
                if (move) R = most_w;
                if (it > 0) {  // the stream's products are complete: its newest scores were issued after them
                    wait_ld(s[0]);
#pragma unroll
                    for (int q = 0; q < HDP / 32; ++q) {
                        ld32(o_tm + 32 * q, s[1]);
                        wait_ld(s[1]);
#pragma unroll
                        for (int j = 0; j < 32; ++j) s[1][j] = __float_as_uint(__uint_as_float(s[1][j]) * fade);
                        st32(o_tm + 32 * q, s[1]);
                    }
                }
            }
            const float raise = R == -INFINITY ? 0.0f : ex2(fminf(ref - R + kLift, 126.0f));
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                vs[g] *= raise;
                if (vs[g] > 3e38f) vs[g] = 3e38f;  // its probabilities are 0 then
            }
            float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                wait_ld(s[q & 1]);
                if (q < 3) ld32(s_tm + 32 * (q + 1), s[(q + 1) & 1]);
                uint32_t out[32];  // hi pairs of 32 slots, then lo pairs
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    float z0 = fmaf(__uint_as_float(s[q & 1][j]), ks[2 * q + j / 16], -ref);
                    float z1 = fmaf(__uint_as_float(s[q & 1][j + 1]), ks[2 * q + j / 16], -ref);
                    if (edge) {
                        if (first + 32 * q + j >= limit) z0 = -INFINITY;
                        if (first + 32 * q + j + 1 >= limit) z1 = -INFINITY;
                    }
                    const float p0 = ex2(z0), p1 = ex2(z1);
                    l0 += p0;
                    l1 += p1;
                    two_terms(p0 * vs[2 * q + j / 16], p1 * vs[2 * q + j / 16], out[j / 2], out[16 + j / 2]);
                }
                st32(s_tm + 32 * q, out);
            }
            l += l0 + l1;
            wait_st();
            tc_before();
            __syncwarp();
            if (lane == 0) dev::mbar_arrive(p_full(x));
        }
    } else if (warp < kMmaWarp) {
        // 128 threads: piece of 16 codes `piece` of rows r0, r0 + kStep, ...
        constexpr int kPieces = HDP / 16, kStep = 128 / kPieces, kLoads = kSlots / kStep;
        const int tid = threadIdx.x - kSoftmaxWarps * 32, piece = tid % kPieces, r0 = tid / kPieces;
        const bool inside = piece * 16 < d;
        const int8_t* kc = c.k_codes + head * c.capacity * d + piece * 16;
        const int8_t* vc = c.v_codes + head * c.capacity * d + piece * 16;
        auto load = [&](const int8_t* from, int tile, uint4 (&w)[kLoads]) {
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int slot = tile * kSlots + r0 + j * kStep;
                w[j] = inside && slot < most ? __ldg(reinterpret_cast<const uint4*>(from + static_cast<int64_t>(slot) * d))
                                             : make_uint4(0, 0, 0, 0);
            }
        };
        auto store = [&](uint32_t tile_at, const uint4 (&w)[kLoads]) {
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int r = r0 + j * kStep;
                uint4 o[2];
                const uint32_t f0 = w[j].x ^ 0x80808080u, f1 = w[j].y ^ 0x80808080u, f2 = w[j].z ^ 0x80808080u, f3 = w[j].w ^ 0x80808080u;
                o[0] = make_uint4(codes_to_half2<0x4140>(f0), codes_to_half2<0x4342>(f0), codes_to_half2<0x4140>(f1),
                                  codes_to_half2<0x4342>(f1));
                o[1] = make_uint4(codes_to_half2<0x4140>(f2), codes_to_half2<0x4342>(f2), codes_to_half2<0x4140>(f3),
                                  codes_to_half2<0x4342>(f3));
                unsigned char* to = smem + tile_at + (piece / 4) * (kSlots * 128);
                const int p2 = piece % 4 * 2, odd = (piece / 4) & 1;  // the two halves of a row in opposite order: no bank conflict
                *reinterpret_cast<uint4*>(to + swizzled(r, p2 + odd)) = odd ? o[1] : o[0];
                *reinterpret_cast<uint4*>(to + swizzled(r, p2 + 1 - odd)) = odd ? o[0] : o[1];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        uint4 kw[kLoads], vw[kLoads];
        load(kc, 0, kw);
        for (int i = 0; i < tiles; ++i) {
            const int y = i & 1;
            load(vc, i, vw);
            if (i >= 2 && !wait_all(k_free(y), (i / 2 - 1) & 1)) break;
            store(S::kK + y * S::kTile, kw);
            if (lane == 0) dev::mbar_arrive(k_full(y));
            if (i + 1 < tiles) load(kc, i + 1, kw);
            if (i >= 2 && !wait_all(v_free(y), (i / 2 - 1) & 1)) break;
            store(S::kV + y * S::kTile, vw);
            if (lane == 0) dev::mbar_arrive(v_full(y));
        }
    } else {
        asm volatile("bar.sync 1, %0;" ::"n"((kSoftmaxWarps + 1) * 32) : "memory");  // the queries are in place
        if (lane == 0) {
            constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(kSlots >> 3) << 17) | (static_cast<uint32_t>(kVecTile >> 4) << 24);
            // the second product's B is MN-major (bit 16)
            constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(HDP >> 3) << 17) |
                                         (static_cast<uint32_t>(kVecTile >> 4) << 24);
            auto scores = [&](int i) {
                const int y = i & 1;
                if (!wait(k_full(y), (i / 2) & 1)) return false;
                tc_after();
#pragma unroll
                for (int s = 0; s < HDP / 16; ++s) {
                    const uint32_t at = (s / 4) * (128 * 128) + (s % 4) * 32;
                    const uint64_t kd = desc_base(base + S::kK + y * S::kTile + at, 16);
                    mma_ss(tmem + y * kSlots, desc_base(base + S::kQ + at, 16), kd, kIdescS, s > 0);
                    mma_ss(tmem + y * kSlots, desc_base(base + S::kQ + S::kTile + at, 16), kd, kIdescS, 1);
                }
                mma_commit(s_full(y));
                mma_commit(k_free(y));
                return true;
            };
            bool go = true;
            for (int i = 0; go && i < min(2, tiles); ++i) go = scores(i);
            for (int i = 0; go && i < tiles; ++i) {
                const int y = i & 1;
                go = wait(v_full(y), (i / 2) & 1) && wait(p_full(y), (i / 2) & 1);
                if (!go) break;
                tc_after();
#pragma unroll
                for (int s = 0; s < kSlots / 16; ++s) {
                    const uint64_t vd = desc_base(base + S::kV + y * S::kTile + s * 2048, kSlots * 128);
                    const uint32_t p = tmem + y * kSlots + (s / 2) * 32 + (s % 2) * 8;
                    mma_ts(tmem + 2 * kSlots + y * HDP, p, vd, kIdescO, i >= 2 || s > 0);
                    mma_ts(tmem + 2 * kSlots + y * HDP, p + 16, vd, kIdescO, 1);
                }
                mma_commit(v_free(y));
                if (i + 2 < tiles) go = scores(i + 2);
            }
            mma_commit(done);
            ok = true;
            wait(done, 0);  // no product is in flight past this point
        }
        __syncwarp();
    }

    // The streams meet: stream 1 leaves its numerators and references, stream 0 adds its own.
    float* const area = reinterpret_cast<float*>(smem + S::kK);            // [dim][vector]
    float* const other = area + HDP * S::kOutPitch;                        // D, l of stream 1
    const uint32_t o_tm = tmem + (static_cast<uint32_t>(row & ~31) << 16) + 2 * kSlots + x * HDP;
    tc_before();
    __syncthreads();
    tc_after();
    if (warp >= 4 && warp < kSoftmaxWarps) {
        other[row] = D;
        other[kVecTile + row] = l;
    }
    __syncthreads();
    float scale = 0.0f;
    if (warp < 4) {
        const float d1 = other[row], l1 = other[kVecTile + row], dm = fmaxf(D, d1);
        const float sum = (l == 0.0f ? 0.0f : l * ex2(D - dm)) + (l1 == 0.0f ? 0.0f : l1 * ex2(d1 - dm));
        other[row] = dm;
        other[kVecTile + row] = 1.0f / sum;
        if (lse != nullptr && row < real)
            lse[(static_cast<int64_t>(b) * a.rows_per_seq + (v0 + row) / group) * a.heads + h * group + (v0 + row) % group] =
                (dm + log2f(sum)) / kLog2e;
    }
    __syncthreads();
    if (warp < kSoftmaxWarps) {
        const float dm = other[row];
        scale = R == -INFINITY ? 0.0f : ex2(R - kLift - dm) * other[kVecTile + row];
        if (l != l) scale = l;
    }
    const bool second = tiles > 1;
#pragma unroll
    for (int turn = 1; turn >= 0; --turn) {
        if (warp < kSoftmaxWarps && x == turn && (turn == 0 || second)) {
#pragma unroll
            for (int q = 0; q < HDP / 32; ++q) {
                uint32_t o[32];
                ld32(o_tm + 32 * q, o);
                wait_ld(o);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    float* to = area + (32 * q + j) * S::kOutPitch + row;
                    const float y = __uint_as_float(o[j]) * scale;
                    *to = turn == 0 && second ? *to + y : y;
                }
            }
        }
        __syncthreads();
    }
    for (int v = warp; v < real; v += kThreads / 32) {
        float* to = a.context + place(v0 + v, static_cast<int64_t>(a.heads) * d);
        for (int i = lane; i < d; i += 32) to[i] = area[i * S::kOutPitch + v];
    }
    tc_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int HDP>
cudaError_t launch(const Kv8Attention& a, int aligned, float* lse, int32_t* err, cudaStream_t s) {
    using S = PromptShape<HDP>;
    const cudaError_t e = cudaFuncSetAttribute(kv8_prompt_kernel<HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    const int64_t vectors = static_cast<int64_t>(a.rows_per_seq) * (a.heads / a.cache.kv_heads);
    const dim3 grid(static_cast<unsigned>((vectors + kVecTile - 1) / kVecTile), a.cache.kv_heads, a.cache.batch);
    return launch_dependent(kv8_prompt_kernel<HDP>, grid, dim3(kThreads), S::kSmem, s, a, aligned, lse, err);
}

}  // namespace

cudaError_t launch_kv8_prompt(const Kv8Attention& a, int aligned, float* lse, int32_t* err, cudaStream_t s) {
    return a.cache.head_dim <= 64 ? launch<64>(a, aligned, lse, err, s) : launch<128>(a, aligned, lse, err, s);
}

}  // namespace kt
