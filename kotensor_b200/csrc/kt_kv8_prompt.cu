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
// Tensor memory holds Q (both terms, the first product's A), the scores of two
// tiles, each replaced in place by its P (a thread owns one vector, a lane of all of
// them; of 32 scores come 16 + 16 columns of hi and lo pairs), and one
// O tile.  Only the B operands, K and V, pass through shared memory: with Q there
// too, the first product alone would take its whole bandwidth.
//   warps 0-3, 4-7  scores -> P of the first, the last 64 slots of a tile; every tile
//                   has its own references, so no tile waits for another's
//   warps 8-11      add each O tile to sums in registers (the tensor cores' fp32
//                   accumulation truncates: over a long run of tiles the error is
//                   five times that of these rounded sums) and write the result
//   warps 12-15     codes -> fp16, K and V tiles in 128-byte swizzled rows of 64 dims
//                   (K-major for the first product, MN-major for the second: the
//                   same bytes, another descriptor)
//   warp 16         issues the products; a warp of its own, since issuing takes as
//                   long as the tensor cores do
//   warp 17         bulk copies of the codes into shared memory, two tiles ahead
// Order of the products: P V of tile i, then Q K^T of tile i + 2; while the second
// runs, O of tile i is read, and tile i + 1 becomes P meanwhile.
//
// References.  A tile's sum l is relative to its largest score D.  The numerators
// carry the values' scales, which may differ by any factor from block to block, so
// they have a reference R of their own, the maximum of score + log2(value scale):
// both terms of P keep 22 bits of what matters to O.
//
// Bound by turns by the products and by the exponentials with the cut of P into terms: a
// tile takes about 3700 clocks, its products 2048.  2 sequences x 509 rows x 32 heads
// of 128 over 1500 to 3508 slots: 102.5 us, 37.6 GFLOP as fp32 counts them, 367 TFLOP/s, or
// 734 with both terms.  (Sixteen softmax warps and two issuing ones 112 us where these
// took 109.)  A CTA spends about 7 us on entering and 3 on leaving.
#include <cuda_fp16.h>

#include <algorithm>

#include "kt_kv8.h"

namespace kt {
namespace {

constexpr int kVecTile = 128;   // query vectors of a CTA (the MMA's M)
constexpr int kSlots = 128;     // slots of a tile (the first product's N, the second's K)
constexpr int kSumWarp = 8;      // first of the four that add up O; before them the softmax warps
constexpr int kConvertWarp = 12; // first of the four that convert
constexpr int kIssueWarp = 16;   // issues the products
constexpr int kCopyWarp = 17;    // copies codes; the two after it do nothing
constexpr int kThreads = 640;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLift = 14.0f;   // numerators are 2^kLift larger: their lo terms stay clear of the subnormals
constexpr float kSlack = 20.0f;  // the sums' reference moves when a tile's passes it by this much
// Registers of a thread at the launch, and of each role's warps, which raise or lower
// theirs (a raise waits for the others' to be freed, so the sum must not grow).
constexpr int kLaunchRegs = 96;
constexpr int kSoftmaxRegs = 120, kSumRegs = 168, kConvertRegs = 48, kIssueRegs = 24;
static_assert(8 * kSoftmaxRegs + 4 * kSumRegs + 4 * kConvertRegs + 4 * kIssueRegs <= 20 * kLaunchRegs, "registers");

// Tensor memory columns.
template <int HDP>
struct PromptShape {
    static constexpr int kBlocks = HDP / 64;              // blocks of 64 dims: 128-byte rows
    static constexpr int kTile = kBlocks * kSlots * 128;  // fp16 tile of 128 rows
    static constexpr int kK = 0, kV = 2 * kTile;
    static constexpr int kRaw = 4 * kTile, kRawTile = kSlots * HDP;  // codes of two K and two V tiles
    static constexpr int kEnd = kRaw + 4 * kRawTile;
    static constexpr int kOutPitch = kVecTile + 1;        // at the end: [dim][vector], over K and V
    // after the tiles: factor and largest component of each query, D, R, l of both halves of
    // four tiles, barriers
    static constexpr int kFactor = kEnd, kTop = kFactor + kVecTile * 4, kStats = kTop + 2 * kVecTile * 4;
    static constexpr int kMeet = kStats + 4 * 4 * kVecTile * 4;         // largest scores of the halves of two tiles
    static constexpr int kBars = kMeet + 4 * kVecTile * 8;
    static constexpr int kSmem = 1024 + kBars + 256;
    static constexpr int kPart = kVecTile * (HDP + 1);    // floats of a split: its results, then logarithms
    static constexpr uint32_t kO = 2 * kSlots, kQ = kO + HDP;  // S of stream x at kSlots * x; Q hi, then lo
    static_assert(HDP * kOutPitch * 4 <= kRaw, "epilogue area");
    static_assert(kSmem <= 232448, "shared memory per CTA");
    static_assert(kQ + HDP <= 512, "tensor memory");
};

__device__ __forceinline__ uint64_t desc_base(uint32_t addr, uint32_t lead) {
    // 128-byte swizzle, atoms of 8 rows 1024 bytes apart, descriptor version 1
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
           (static_cast<uint64_t>(2) << 61);
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
// The same for 16 columns, complete on return.
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
    static_assert(N <= kLaunchRegs && N % 8 == 0 && N >= 24, "can only lower");
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void more_registers() {
    static_assert(N >= kLaunchRegs && N % 8 == 0 && N <= 256, "can only raise");
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
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
// Four codes as fp16 pairs {0, 2} and {1, 3}: a mask leaves every other byte, an
// exclusive or makes it 0x64xx with the sign bit flipped, 1024 + code + 128, and
// 1152 is taken off.  (Masks run at twice the rate of byte permutations; the tiles'
// dims are in the order 0, 2, 1, 3 of every four, and so are the queries'.)
__device__ __forceinline__ uint2 codes_to_half(uint32_t w) {
    const __half2 offset = __half2half2(__ushort_as_half(0x6480));
    const uint32_t even = (w & 0x00ff00ffu) ^ 0x64806480u, odd = ((w >> 8) & 0x00ff00ffu) ^ 0x64806480u;
    return make_uint2(h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&even), offset)),
                      h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&odd), offset)));
}
// Byte offset of 16-byte piece `piece` (of 64 dims: 8) of row `row` in a swizzled block.
__device__ __forceinline__ uint32_t swizzled(int row, int piece) {
    return static_cast<uint32_t>(row * 128 + ((piece ^ (row & 7)) << 4));
}

// Waits for phase `parity` of `bar`; false after some seconds.  The hardware holds a
// try for about a hundred cycles; reading a clock between tries, as the bounded wait
// of kt_device.cuh does, or giving the try a longer time (which becomes a loop of
// sleeps) took a third of the SM's issue slots from the warps that work.
__device__ __forceinline__ bool wait_counted(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 25); ++i)
        if (dev::mbar_try_wait(bar, parity)) return true;
    return false;
}
// Two fp32 operations at a time.
__device__ __forceinline__ uint64_t pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& x, float& y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

// Scores of 64 slots of a tile -> their P in place, for the vector of this thread:
// first slot `first`, S at tensor memory address s_tm; P's hi terms of 32 slots lie in
// the first 16 columns of theirs, the lo terms in the last.  Lane g of the warp has
// the scales of slots first + 16 g .. in k_scale, v_scale.  The thread with the
// vector's other 64 slots is in the warp that shares barrier `bar`; their largest
// scores meet in mine, other; false if that warp gave up (it left NaN there, as no largest
// score is).  kEdge: some vector of the warp does not see all of
// the slots; this one sees those below `limit`.  The loops stay rolled and the scores
// are read twice: unrolled, the roles' code did not fit the instruction caches, and
// waiting for instructions was the longest of all stalls.
template <bool kEdge>
__device__ __forceinline__ bool scores_to_p(uint32_t s_tm, int first, int limit, float factor, float k_scale,
                                            float v_scale, float2* mine, const float2* other, int bar, float& D,
                                            float& l, float& R) {
    // a block the vector does not see has no scale, whatever is there
    auto k_of = [&](int g) {
        const float k = __shfl_sync(0xffffffffu, k_scale, g) * factor;
        return kEdge && first + 16 * g >= limit ? 0.0f : k;
    };
    auto v_of = [&](int g) {
        const float v = __shfl_sync(0xffffffffu, v_scale, g);
        return kEdge && first + 16 * g >= limit ? 0.0f : v;
    };
    D = R = -INFINITY;
#pragma unroll 1
    for (int g = 0; g < 4; ++g) {
        uint32_t s[16];
        const float k = k_of(g), v = __log2f(v_of(g));
        ld16(s_tm + 16 * g, s);
        float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = __uint_as_float(s[j + i]);
                if (kEdge && first + 16 * g + j + i >= limit) x[i] = -INFINITY;
            }
            m[0] = max3(m[0], x[0], x[1]);
            m[1] = max3(m[1], x[2], x[3]);
        }
        float top = fmaxf(m[0], m[1]);
        top = top == -INFINITY ? top : top * k;
        D = fmaxf(D, top);
        R = fmaxf(R, top + v);
    }
    *mine = make_float2(D, R);
    asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");
    const float2 there = *other;
    if (__any_sync(0xffffffffu, there.x != there.x)) return false;
    D = fmaxf(D, there.x);
    R = fmaxf(R, there.y);
    const float ref = D == -INFINITY ? 0.0f : D;
    const float raise = R == -INFINITY ? 0.0f : ex2(fminf(ref - R + kLift, 126.0f));
    const uint64_t less = pair(-ref, -ref);
    uint64_t sum = pair(0.0f, 0.0f);
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        uint32_t lo[2][8];  // kept until both halves of these 32 scores have been read
        uint32_t hi[2][8];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            uint32_t s[16];
            ld16(s_tm + 32 * h + 16 * g, s);
            const float k = k_of(2 * h + g);
            float v = v_of(2 * h + g) * raise;
            if (v > 3e38f) v = 3e38f;  // its probabilities are 0 then
            const uint64_t kk = pair(k, k), vv = pair(v, v);
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                float z0, z1;
                unpair(fma2(pair(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), kk, less), z0, z1);
                if (kEdge) {
                    if (first + 32 * h + 16 * g + j >= limit) z0 = -INFINITY;
                    if (first + 32 * h + 16 * g + j + 1 >= limit) z1 = -INFINITY;
                }
                const uint64_t p = pair(ex2(z0), ex2(z1));
                sum = add2(sum, p);
                const uint64_t n = mul2(p, vv);
                float n0, n1, r0, r1;
                unpair(n, n0, n1);
                const __half2 high = __floats2half2_rn(n0, n1);
                const float2 back = __half22float2(high);
                unpair(add2(n, pair(-back.x, -back.y)), r0, r1);
                hi[g][j / 2] = h2_bits(high);
                lo[g][j / 2] = h2_bits(__floats2half2_rn(r0, r1));
            }
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            st8(s_tm + 32 * h + 8 * g, hi[g]);
            st8(s_tm + 32 * h + 16 + 8 * g, lo[g]);
        }
    }
    float s0, s1;
    unpair(sum, s0, s1);
    l = s0 + s1;
    return true;
}

template <int HDP>
__global__ void __launch_bounds__(kThreads, 1) kv8_prompt_kernel(Kv8Attention a, int aligned, int splits,
                                                                 float* __restrict__ parts, float* __restrict__ lse,
                                                                 int32_t* __restrict__ err) {
    using S = PromptShape<HDP>;
    dev::pdl_wait();
    const Kv8& c = a.cache;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, d = c.head_dim;
    const int b = blockIdx.z, h = blockIdx.y;
    const int vt = gridDim.x / splits - 1 - blockIdx.x / splits;  // the rows that see most first
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
    // the CTA's tiles: part `split` of those its vectors see, numbered from `from`
    const int all_tiles = (most + kSlots - 1) / kSlots, split = blockIdx.x % splits;
    const int from = split * all_tiles / splits, tiles = (split + 1) * all_tiles / splits - from;
    // with splits, each leaves its result and the logarithms of its sums in its place
    float* const part = parts + ((static_cast<int64_t>(b) * c.kv_heads + h) * (gridDim.x / splits) + vt) * splits * S::kPart +
                        static_cast<int64_t>(split) * S::kPart;
    if (tiles == 0) {
        for (int v = threadIdx.x; v < kVecTile; v += kThreads) part[kVecTile * HDP + v] = -INFINITY;
        dev::pdl_launch_dependents();
        return;
    }

    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = dev::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* const smem = smem_raw + (base - raw);
    float* const q_factor = reinterpret_cast<float*>(smem + S::kFactor);
    float* const q_top = reinterpret_cast<float*>(smem + S::kTop);
    float* const stats = reinterpret_cast<float*>(smem + S::kStats);  // [tile % 4][D, R, l, l][vector]
    float2* const meet = reinterpret_cast<float2*>(smem + S::kMeet);  // [tile % 2][half][vector]
    const uint32_t bars = base + S::kBars;
    auto k_full = [&](int x) { return bars + 8 * x; };
    auto k_free = [&](int x) { return bars + 16 + 8 * x; };
    auto v_full = [&](int x) { return bars + 32 + 8 * x; };
    auto v_free = [&](int x) { return bars + 48 + 8 * x; };
    auto s_full = [&](int x) { return bars + 64 + 8 * x; };
    auto p_full = [&](int x) { return bars + 80 + 8 * x; };
    const uint32_t o_full = bars + 96, o_free = bars + 104;
    auto raw_full = [&](int v, int x) { return bars + 112 + 16 * v + 8 * x; };  // v: 0 keys, 1 values
    auto raw_free = [&](int v, int x) { return bars + 144 + 16 * v + 8 * x; };
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kBars + 176);
    if (threadIdx.x == 0) {
        for (int x = 0; x < 2; ++x) {
            dev::mbar_init(k_full(x), 4);
            dev::mbar_init(k_free(x), 1);
            dev::mbar_init(v_full(x), 4);
            dev::mbar_init(v_free(x), 1);
            dev::mbar_init(s_full(x), 1);
            dev::mbar_init(p_full(x), 8);
            dev::mbar_init(raw_full(0, x), 1);
            dev::mbar_init(raw_full(1, x), 1);
            dev::mbar_init(raw_free(0, x), 4);
            dev::mbar_init(raw_free(1, x), 4);
        }
        dev::mbar_init(o_full, 1);
        dev::mbar_init(o_free, 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssueWarp) {
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
        if (!wait_counted(bar, parity)) {
            ok = false;
            atomicOr(err, 1);
        }
        return ok;
    };
    auto wait_all = [&](uint32_t bar, uint32_t parity) {  // a warp: its lanes go on, or give up, together
        return __all_sync(0xffffffffu, wait(bar, parity));
    };
    const int row = (warp % 4) * 32 + lane;  // the vector, and lane of tensor memory, of a thread
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp % 4) << 21);

    if (warp < kSumWarp) {
        more_registers<kSoftmaxRegs>();
        const int x = warp / 4;
        {
            // Queries: scaled by a power of two to at most 1, in two terms; a negative scale
            // turns their sign.  Warps 0-3 take the first half of the dims, 4-7 the second.
            constexpr int kHalf = HDP / 2;
            const float* q = a.q + place(v0 + row, a.q_stride) + x * kHalf;
            float f[kHalf];
            uint32_t top = 0;  // the largest exponent, by the bits of |q|; NaN counts as infinity
#pragma unroll
            for (int i = 0; i < kHalf; i += 4) {
                f[i] = f[i + 1] = f[i + 2] = f[i + 3] = 0.0f;
                if (row < real && x * kHalf + i < d) {
                    if (aligned & 1) {
                        const float4 t = *reinterpret_cast<const float4*>(q + i);
                        f[i] = t.x, f[i + 1] = t.y, f[i + 2] = t.z, f[i + 3] = t.w;
                    } else {
                        f[i] = q[i], f[i + 1] = q[i + 1], f[i + 2] = q[i + 2], f[i + 3] = q[i + 3];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kHalf; ++i) top = max(top, min(__float_as_uint(f[i]) & 0x7fffffffu, 0x7f800000u));
            q_top[x * kVecTile + row] = __uint_as_float(top);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            top = max(top, __float_as_uint(q_top[(1 - x) * kVecTile + row]));
            const int e = min(max(static_cast<int>(top >> 23) - 126, -126), 126);
            float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            if (a.scale < 0.0f) down = -down;
            if (x == 0) q_factor[row] = fabsf(a.scale) * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
            for (int q = 0; q < kHalf; q += 32) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; i += 2) {  // the tiles' order of dims
                    two_terms(f[q + 2 * i] * down, f[q + 2 * i + 2] * down, hi[i], lo[i]);
                    two_terms(f[q + 2 * i + 1] * down, f[q + 2 * i + 3] * down, hi[i + 1], lo[i + 1]);
                }
                st16(lanes + S::kQ + (x * kHalf + q) / 2, hi);
                st16(lanes + S::kQ + HDP / 2 + (x * kHalf + q) / 2, lo);
            }
            wait_st();
            tc_before();
            asm volatile("bar.sync 2, 288;" ::: "memory");  // with the issuing warp: the queries are in place
        }
        const float factor = q_factor[row];
        // (lanes without a vector compute something that nobody reads)
        const int limit = row < real ? min(held + (v0 + row) / group + 1, seen) : most;
        const float* k_scales = c.k_scales + head * (c.capacity / c.block);
        const float* v_scales = c.v_scales + head * (c.capacity / c.block);
        for (int i = 0; i < tiles; ++i) {
            const int y = i & 1, first = (from + i) * kSlots + 64 * x, at = first + 16 * (lane % 4);
            const float ks = at < most ? k_scales[at / c.block] : 0.0f, vs = at < most ? v_scales[at / c.block] : 0.0f;
            float2* const mine = meet + (2 * y + x) * kVecTile + row;
            const float2* const other = meet + (2 * y + 1 - x) * kVecTile + row;
            const int bar = 4 + warp % 4;
            if (!wait_all(s_full(y), (i / 2) & 1)) {  // the other half's warp may have seen it: not left waiting
                *mine = make_float2(__uint_as_float(0x7fc00000u), 0.0f);
                asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");
                break;
            }
            tc_after();
            const uint32_t s_tm = lanes + y * kSlots + 64 * x;
            float D, l, R;
            if (!(__any_sync(0xffffffffu, first + 64 > limit)
                      ? scores_to_p<true>(s_tm, first, limit, factor, ks, vs, mine, other, bar, D, l, R)
                      : scores_to_p<false>(s_tm, first, limit, factor, ks, vs, mine, other, bar, D, l, R)))
                break;
            float* const to = stats + (i % 4) * 4 * kVecTile + row;
            if (x == 0) to[0] = D, to[kVecTile] = R;
            to[(2 + x) * kVecTile] = l;
            wait_st();
            tc_before();
            __syncwarp();
            if (lane == 0) dev::mbar_arrive(p_full(y));
        }
    } else if (warp >= kIssueWarp) {
        fewer_registers<kIssueRegs>();
        constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(kSlots >> 3) << 17) | (static_cast<uint32_t>(kVecTile >> 4) << 24);
        // the second product's B is MN-major (bit 16)
        constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(HDP >> 3) << 17) |
                                     (static_cast<uint32_t>(kVecTile >> 4) << 24);
        auto scores = [&](int i) {  // the small terms first: the accumulator's truncation is relative to its value
            const int y = i & 1;
            if (!wait(k_full(y), (i / 2) & 1)) return;
            tc_after();
            const uint64_t kd = desc_base(base + S::kK + y * S::kTile, 16);
#pragma unroll
            for (int s = 0; s < HDP / 8; ++s) {
                const int k = s % (HDP / 16), term = s < HDP / 16 ? 1 : 0;
                mma_ts(tmem + y * kSlots, tmem + S::kQ + term * (HDP / 2) + 8 * k, kd + ((k / 4) * (128 * 128) + (k % 4) * 32) / 16,
                       kIdescS, s > 0);
            }
            mma_commit(s_full(y));
            mma_commit(k_free(y));
        };
        if (warp == kIssueWarp) {
            asm volatile("bar.sync 2, 288;" ::: "memory");  // the queries are in place
            tc_after();
            if (lane == 0) {
                for (int i = 0; i < min(2, tiles); ++i) scores(i);
                for (int i = 0; ok && i < tiles; ++i) {
                    const int y = i & 1;
                    if (!wait(v_full(y), (i / 2) & 1) || !wait(p_full(y), (i / 2) & 1) || (i > 0 && !wait(o_free, (i - 1) & 1))) break;
                    tc_after();
                    const uint64_t vd = desc_base(base + S::kV + y * S::kTile, kSlots * 128);
#pragma unroll
                    for (int s = 0; s < kSlots / 8; ++s) {
                        const int k = s % (kSlots / 16), term = s < kSlots / 16 ? 1 : 0;
                        mma_ts(tmem + S::kO, tmem + y * kSlots + (k / 2) * 32 + (k % 2) * 8 + term * 16, vd + k * 2048 / 16,
                               kIdescO, s > 0);
                    }
                    mma_commit(o_full);
                    mma_commit(v_free(y));
                    if (i + 2 < tiles) scores(i + 2);
                }
            }
            __syncwarp();
        } else if (warp == kCopyWarp) {
            if (lane == 0) {
                int sent[2] = {0, 0};
                auto copy = [&](int v, int i) {
                    const int y = i & 1;
                    if (i >= 2 && !wait(raw_free(v, y), (i / 2 - 1) & 1)) return;
                    // (slots past the last one seen have some code: their scores are masked, their P is 0)
                    const int slot = (from + i) * kSlots;
                    const uint32_t bytes = static_cast<uint32_t>(min(kSlots, c.capacity - slot) * d);
                    const int8_t* codes = (v ? c.v_codes : c.k_codes) + (head * c.capacity + slot) * d;
                    dev::mbar_expect_tx(raw_full(v, y), bytes);
                    dev::bulk_load(base + S::kRaw + (2 * v + y) * S::kRawTile, codes, bytes, raw_full(v, y));
                    sent[v] = i + 1;
                };
                copy(0, 0);
                if (tiles > 1) copy(0, 1);
                for (int i = 0; ok && i < tiles; ++i) {
                    copy(1, i);
                    if (ok && i + 2 < tiles) copy(0, i + 2);
                }
                // no copy is in flight past this point, also where a wait has given up
#pragma unroll
                for (int v = 0; v < 2; ++v)
                    for (int i = max(0, sent[v] - 2); i < sent[v]; ++i)
                        if (!wait_counted(raw_full(v, i & 1), (i / 2) & 1)) atomicOr(err, 1);
            }
            __syncwarp();
        }
    } else if (warp >= kConvertWarp) {
        fewer_registers<kConvertRegs>();
        // 128 threads: piece of 16 codes `piece` of rows r0, r0 + kStep, ...; eight
        // neighbours have four pieces of two adjacent rows, whose 16-byte stores fall in
        // different banks
        constexpr int kPieces = HDP / 16, kStep = 128 / kPieces, kLoads = kSlots / kStep;
        const int tid = threadIdx.x - kConvertWarp * 32, piece = tid % 4 + tid / 8 % (kPieces / 4) * 4;
        const int r0 = tid / 4 % 2 + tid / (2 * kPieces) * 2;
        auto convert = [&](int v, int i, uint32_t tile_at) {  // keys or values of tile i; false: gave up
            const int y = i & 1;
            if (!wait_all(raw_full(v, y), (i / 2) & 1)) return false;
            const unsigned char* from = smem + S::kRaw + (2 * v + y) * S::kRawTile + piece * 16;
#pragma unroll 2
            for (int j = 0; j < kLoads; ++j) {
                const int r = r0 + j * kStep;
                const uint4 c4 = piece * 16 < d ? *reinterpret_cast<const uint4*>(from + r * d) : make_uint4(0, 0, 0, 0);
                const uint2 h0 = codes_to_half(c4.x), h1 = codes_to_half(c4.y), h2 = codes_to_half(c4.z), h3 = codes_to_half(c4.w);
                unsigned char* to = smem + tile_at + y * S::kTile + (piece / 4) * (kSlots * 128);
                *reinterpret_cast<uint4*>(to + swizzled(r, piece % 4 * 2)) = make_uint4(h0.x, h0.y, h1.x, h1.y);
                *reinterpret_cast<uint4*>(to + swizzled(r, piece % 4 * 2 + 1)) = make_uint4(h2.x, h2.y, h3.x, h3.y);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                dev::mbar_arrive(raw_free(v, y));
                dev::mbar_arrive(v == 0 ? k_full(y) : v_full(y));
            }
            return true;
        };
        // K(0), K(1), V(0), K(2), V(1), ...: the products need K(i + 2) right after V(i)
        bool go = convert(0, 0, S::kK);
        if (go && tiles > 1) go = convert(0, 1, S::kK);
        for (int i = 0; go && i < tiles; ++i) {
            const int y = i & 1;
            if (i >= 2 && !wait_all(v_free(y), (i / 2 - 1) & 1)) break;
            if (!convert(1, i, S::kV)) break;
            if (i + 2 >= tiles) continue;
            if (!wait_all(k_free(y), (i / 2) & 1)) break;
            go = convert(0, i + 2, S::kK);
        }
    } else {
        more_registers<kSumRegs>();
        uint64_t o[HDP / 2];
        float D = -INFINITY, l = 0.0f, R = -INFINITY;
#pragma unroll
        for (int j = 0; j < HDP / 2; ++j) o[j] = 0;
        for (int i = 0; i < tiles; ++i) {
            const int y = i & 1;
            // Every warp has seen tile i's P before it gives up tile i - 1's O, and the next
            // product into O waits for both: no barrier runs two phases ahead of a warp.
            if (!wait_all(p_full(y), (i / 2) & 1)) break;
            if (i > 0 && lane == 0) dev::mbar_arrive(o_free);
            if (!wait_all(o_full, i & 1)) break;
            tc_after();
            const float* tile = stats + (i % 4) * 4 * kVecTile + row;
            const float tD = tile[0], tR = tile[kVecTile], tl = tile[2 * kVecTile] + tile[3 * kVecTile];
            const float top = fmaxf(D, tD);
            l = (l == 0.0f ? 0.0f : l * ex2(D - top)) + (tl == 0.0f ? 0.0f : tl * ex2(tD - top));
            D = top;
            const bool move = tR > R + kSlack || (R == -INFINITY && tR > R);
            if (__any_sync(0xffffffffu, move)) {
                const float fade = !move ? 1.0f : R == -INFINITY ? 0.0f : ex2(R - tR);
                if (move) R = tR;
#pragma unroll
                for (int j = 0; j < HDP / 2; ++j) o[j] = mul2(o[j], pair(fade, fade));
            }
            const float by = tR == -INFINITY ? 0.0f : ex2(tR - R);
            const uint64_t gain = pair(by, by);
#pragma unroll
            for (int q = 0; q < HDP / 32; ++q) {
                uint32_t part[32];
                ld32(lanes + S::kO + 32 * q, part);
                wait_ld(part);
#pragma unroll
                for (int j = 0; j < 32; j += 2)
                    o[16 * q + j / 2] = fma2(pair(__uint_as_float(part[j]), __uint_as_float(part[j + 1])), gain, o[16 * q + j / 2]);
            }
            tc_before();
            __syncwarp();
        }
        // every product is complete (the last o_full came after all of them): K and V are free
        if (splits > 1) part[kVecTile * HDP + row] = D + log2f(l);
        else if (lse != nullptr && row < real)
            lse[(static_cast<int64_t>(b) * a.rows_per_seq + (v0 + row) / group) * a.heads + h * group + (v0 + row) % group] =
                (D + log2f(l)) / kLog2e;
        const float scale = l != l ? l : R == -INFINITY ? 0.0f : ex2(R - kLift - D) / l;
        float* const area = reinterpret_cast<float*>(smem);  // [dim][vector]
#pragma unroll
        for (int j = 0; j < HDP; j += 2) {
            float y0, y1;
            unpair(o[j / 2], y0, y1);
            const int dim = j / 4 * 4 + j / 2 % 2;  // columns j, j + 1 are dims dim, dim + 2
            area[dim * S::kOutPitch + row] = y0 * scale;
            area[(dim + 2) * S::kOutPitch + row] = y1 * scale;
        }
        asm volatile("bar.sync 3, 128;" ::: "memory");
        // Each lane works out where one of the warp's 32 vectors goes; then four vectors at a time, so that the
        // loads and stores of one do not wait for another's (one vector at a time took 5 to 7 us a CTA, this 1.6 to 2.3).
        const int first = warp - kSumWarp, own = first + 4 * lane;
        float* const base = splits > 1 ? part : a.context;
        const int64_t at = splits > 1 ? static_cast<int64_t>(own) * HDP
                           : own < real ? place(v0 + own, static_cast<int64_t>(a.heads) * d)
                                        : 0;
#pragma unroll 1
        for (int n = 0; first + 4 * n < real; n += 4) {
            float y[4][HDP / 32];
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < HDP / 32; ++i) y[k][i] = area[(32 * i + lane) * S::kOutPitch + first + 4 * (n + k)];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float* const to = base + __shfl_sync(0xffffffffu, at, n + k);
                if (first + 4 * (n + k) < real)
#pragma unroll
                    for (int i = 0; i < HDP / 32; ++i)
                        if (32 * i + lane < d) to[32 * i + lane] = y[k][i];
            }
        }
    }
    tc_before();
    __syncthreads();
    if (warp == kIssueWarp) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// The splits of a vector's slots: a warp to a vector, results weighted by their sums.
template <int HDP>
__global__ void __launch_bounds__(256) kv8_prompt_merge_kernel(Kv8Attention a, int splits, const float* __restrict__ parts,
                                                               float* __restrict__ lse) {
    using S = PromptShape<HDP>;
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const Kv8& c = a.cache;
    const int b = blockIdx.z, h = blockIdx.y, v = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32, d = c.head_dim;
    const int group = a.heads / c.kv_heads, rows = kv8_rows(a.counts, b, a.rows_per_seq);
    if (v >= rows * group) return;
    const int tiles = (a.rows_per_seq * group + kVecTile - 1) / kVecTile;
    const float* part = parts + ((static_cast<int64_t>(b) * c.kv_heads + h) * tiles + v / kVecTile) * splits * S::kPart;
    const int at = v % kVecTile;
    float top = -INFINITY, sum = 0.0f, y[HDP / 32] = {};
    for (int s = 0; s < splits; ++s) top = fmaxf(top, part[s * S::kPart + kVecTile * HDP + at]);
    for (int s = 0; s < splits; ++s) {
        const float z = part[s * S::kPart + kVecTile * HDP + at];
        if (z == -INFINITY) continue;
        const float by = ex2(z - top);
        sum += by;
#pragma unroll
        for (int i = 0; i < HDP / 32; ++i)
            if (lane + 32 * i < d) y[i] = fmaf(by, part[s * S::kPart + at * HDP + lane + 32 * i], y[i]);
    }
    const int64_t row = static_cast<int64_t>(b) * a.rows_per_seq + v / group;
    const int head = h * group + v % group;
#pragma unroll
    for (int i = 0; i < HDP / 32; ++i)
        if (lane + 32 * i < d) a.context[row * a.heads * d + static_cast<int64_t>(head) * d + lane + 32 * i] = y[i] / sum;
    if (lse != nullptr && lane == 0) lse[row * a.heads + head] = (top + log2f(sum)) / kLog2e;
}

template <int HDP>
cudaError_t launch(const Kv8Attention& a, int aligned, float* parts, float* lse, int32_t* err, cudaStream_t s) {
    using S = PromptShape<HDP>;
    static std::atomic<uint64_t> allowed{0};
    cudaError_t e = allow_shared(kv8_prompt_kernel<HDP>, S::kSmem, allowed);
    if (e != cudaSuccess) return e;
    static const int regs = [] {  // what the compiler gave the kernel has to be what the roles share out
        cudaFuncAttributes f{};
        return cudaFuncGetAttributes(&f, kv8_prompt_kernel<HDP>) == cudaSuccess ? f.numRegs : -1;
    }();
    if (regs != kLaunchRegs) return cudaErrorInvalidConfiguration;
    const int64_t vectors = static_cast<int64_t>(a.rows_per_seq) * (a.heads / a.cache.kv_heads);
    const int64_t tiles = (vectors + kVecTile - 1) / kVecTile;
    // Too few CTAs for the card: each vector tile's slots in parts.  (4 sequences of 8 key/value
    // heads, 60 rows of 4 heads each, 4000 slots: 64 CTAs 80 us, 128 of half the slots 53 us.)
    const int splits = kv8_prompt_splits(a.cache.batch, a.rows_per_seq, a.heads, a.cache.kv_heads, a.cache.capacity);
    const dim3 grid(static_cast<unsigned>(tiles * splits), a.cache.kv_heads, a.cache.batch);
    e = launch_dependent(kv8_prompt_kernel<HDP>, grid, dim3(kThreads), S::kSmem, s, a, aligned, splits, parts, lse, err);
    if (e == cudaSuccess && splits > 1)
        e = launch_dependent(kv8_prompt_merge_kernel<HDP>, dim3(static_cast<unsigned>((vectors + 7) / 8), a.cache.kv_heads, a.cache.batch),
                             dim3(256), 0, s, a, splits, static_cast<const float*>(parts), lse);
    return e;
}

}  // namespace

int kv8_prompt_splits(int32_t batch, int32_t rows_per_seq, int32_t heads, int32_t kv_heads, int32_t capacity) {
    const int64_t vectors = static_cast<int64_t>(rows_per_seq) * (heads / kv_heads);
    const int64_t ctas = static_cast<int64_t>(batch) * kv_heads * ((vectors + kVecTile - 1) / kVecTile);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kPromptCtas / ctas, 16, (capacity + kSlots - 1) / kSlots})));
}

size_t kv8_prompt_bytes(int32_t head_dim) {
    return static_cast<size_t>(kPromptCtas) * (head_dim <= 64 ? PromptShape<64>::kPart : PromptShape<128>::kPart) * sizeof(float);
}

cudaError_t launch_kv8_prompt(const Kv8Attention& a, int aligned, float* parts, float* lse, int32_t* err, cudaStream_t s) {
    return a.cache.head_dim <= 64 ? launch<64>(a, aligned, parts, lse, err, s) : launch<128>(a, aligned, parts, lse, err, s);
}

}  // namespace kt
