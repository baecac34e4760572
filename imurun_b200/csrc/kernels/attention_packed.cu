// attention_packed.cu — causal attention of packed prompts of different lengths
// on the 5th-generation tensor cores.
//
//   O_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c s_ij - m_i),  s_ij = q_i . k_j,
// over the keys j that row i sees, c = scale log2(e), m_i a running reference.
//
// A tile is 128 MMA rows: R = 128 / G consecutive rows of one sequence times the
// G query heads of one kv head, so grouped heads share a tile whatever G is and
// short prompts still fill it. A job is two neighbouring tiles (2 R rows), which
// share every key and value tile. A CTA an SM takes its part of the jobs, longest
// first; every role goes from one job to the next by itself, so loads and scores
// of the next job run under the last weights and the output of this one.
// Warps:
//   0..3, 4..7  softmax of tile 0 and 1, a thread a row: scores from tensor
//               memory, mask, row maximum, weights in 16 bits back over the
//               scores' columns; at the end the rows of out;
//   8           the MMAs: S_x = Q_x K_j^T (both from shared memory), then
//               O_x += P_x V_j with P_x from tensor memory. While one tile's
//               warps form weights, the tensor core works for the other;
//   9           TMA: Q, then K and V tiles of BK rows through a ring;
//   10          tiles of V in which some row does not see some key: values that
//               are not finite are taken out before the product (0 x inf is
//               NaN) and their rows noted; rows that do see them add them at
//               the end, from the noted rows alone;
//   11          looks up the jobs to come.
// Tensor memory: S0 S1 (128 columns each), O0 O1. Key tiles have 128 rows or 64.
// With 128 a tile's scores take its 128 columns, P the first 64 of them, and the
// scores of the next keys wait for the product: S0 S1 | O0 S0 O1 S1 | O0 S0 ..
// With 64 there are two places, so scores are ahead of the weights by one tile
// and less is computed beyond the diagonal; but a product of 64 columns takes
// the tensor core longer than half of one of 128, and each step has its fixed
// part. Measured with D = 64, 96, 128 (us, tiles of 64 against 128): 64 prompts of
// 0-300 rows 27 - 31, 33 - 35, 33 - 37; 16 of 600-1000 96 - 94, 113 - 117,
// 117 - 127; 16 of 100-2047 174 - 168, 205 - 204, 215 - 223; one of 8192
// 213 - 191, 236 - 211, 270 - 225. So the mean length decides, at 10 D rows. Where
// the jobs are no more than the SMs the longest one is all the time, and 128 it is:
// one prompt of 512 rows 18 - 17, 20 - 18, 20.5 - 19.5 (those with cold caches).
//
// The reference m_i is raised only when a tile's maximum exceeds it by 2^kSlack,
// so the accumulator is rescaled a few times a row, not once a tile. Weights are
// rounded to the values' type for the product, their sum is not: relative errors
// of 2^-11 or 2^-8 that differ from key to key and average out. f16's range is
// small, so there all weights are 2^11 times as large (at most 2^15): they keep
// their bits down to 2^-25 of the row's largest, and those below 2^-36 are lost,
// for a slack of 2^4 instead of 2^8, which takes 0.5 us of 22 at 64 prompts of
// 0-300 rows and nothing of longer ones.
//
// What bounds it: long prompts the tensor core under the power limit. One of
// 16384 rows, 64 heads in 8 groups, D = 128: 3.84 ms, 1.15 PFLOP/s; the same
// kernel without its softmax takes 3.14 ms, which is the rate of a large matrix
// product over as long a time. The tensor core is fed 1140 cycles a tile and 128
// keys where 1024 would do (shared memory gives the scores' two operands at just
// its rate) and waits 340 for weights. Shorter prompts: the change from job to
// job, some 9000 cycles of 26000 at 1000 rows (weights and output of the first
// and last tiles, which nothing else covers), and 5 us for launch and first loads.
// Tried and slower: a warpgroup of its own for the output (286 us against 247 at
// 16 of 100-2047 rows), two threads a row (251), weights handed over in four
// parts, part of the exponentials on the FMA pipe, two warps that issue MMAs.
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>
#include <mutex>

#include "kv4.cuh"
#include "launch.cuh"
#include "umma.cuh"

namespace fb {
namespace pk {

constexpr int kHalf = 128 * 128;         // 128 rows x 64 values of 16 bits: one SW128 box
constexpr int kSoft = 256, kThreads = kSoft + 128;
constexpr int NJ = 4;                    // jobs looked up ahead
// weights are 2^(c s - m + kUp), up to 2^(kSlack + kUp)
template <class E> struct Range { static constexpr float kSlack = 8.0f, kUp = 0.0f; };
template <> struct Range<__half> { static constexpr float kSlack = 4.0f, kUp = 11.0f; };

// BK keys a tile, NB = 128 / BK places of a tile's scores in tensor memory, NS ring places of a V and a K tile
template <int D, int BK>
struct Smem {
    static constexpr int NB = 128 / BK, NS = 2 * NB, half = BK * 128;
    static constexpr int halves = (D + 63) / 64;
    static constexpr int qtile = halves * kHalf, tile = halves * half;   // one Q tile; one K or V tile
    static constexpr int place = 2 * tile;                 // V_j and, behind it, K_{j+NB}
    static constexpr int ring = 2 * qtile, out = ring + NS * place, bar = out + 8 * 4096;   // out: 32 rows x 128 bytes a warp
    enum { B_Q = 0, B_QFREE, B_FULL, B_EMPTY = B_FULL + NS, B_CLEAN = B_EMPTY + NS, B_S = B_CLEAN + NS, B_P = B_S + 4, B_O = B_P + 4,
           B_END = B_O + 2, B_DRAIN = B_END + 2, B_JOB, B_TAKEN = B_JOB + NJ, B_COUNT = B_TAKEN + NJ };
    // rows of a job's masked tiles, a bit each: up to 255 neighbouring keys at either end
    static constexpr int words = 2 * ((254 + BK - 1) / BK + 1) * (BK / 32);
    static_assert(words <= 32, "a lane clears a word");
    static constexpr int bytes = bar + 8 * B_COUNT + 48 + 16 * NJ + 4 * 2 * NJ * words + 1024;
    static_assert(bytes <= 232448, "shared memory");
};

// The tensor core's additions cut off, so an accumulator loses, at every product of 16 keys, some share of what it holds: 2e-7
// as measured (results of 131072 keys were 7.5e-4 too small and of 2^20 5.7e-3, for 64, 96 and 128 dimensions, f16 and bf16,
// with values of one sign). The weights' own sum is cut by the same share, so that the division takes it out: 5e-5 and 8e-5 are left.
constexpr float kCut = 3.375f / (1 << 24);

struct Job {
    int s0, s1, r0;   // the sequence's rows, the first row of the job's tiles
};
// Key tiles [from[x], to[x]) of a job's tile x, counted from the sequence's start; `masked` where some row of the job does not
// see some key of the tile.
template <int BK>
struct Keys {
    int lo[2], hi[2], from[2], to[2], j0, j1, upper, lower;
    __device__ __forceinline__ Keys(const Job& job, int R, int w) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            lo[x] = job.r0 + x * R - job.s0;
            hi[x] = min(lo[x] + R, job.s1 - job.s0) - 1;   // rows of the tile
            from[x] = w > 0 ? max(0, lo[x] - w + 1) / BK : 0;
            to[x] = lo[x] < job.s1 - job.s0 ? hi[x] / BK + 1 : 0;
        }
        j0 = from[0];
        j1 = max(to[0], to[1]);
        upper = (lo[0] + 1) / BK;                                     // from here on keys past the first row
        const int out = (to[1] ? hi[1] : hi[0]) - w;
        lower = w > 0 && out >= 0 ? out / BK : -1;                    // up to here keys before the last row's window
    }
    __device__ __forceinline__ bool active(int x, int j) const { return j >= from[x] && j < to[x]; }
    __device__ __forceinline__ bool masked(int j) const { return j >= upper || j <= lower; }
    // how many masked tiles come before the masked tile j, and the next masked tile
    __device__ __forceinline__ int place(int j) const { return j - j0 - (j > lower ? max(0, upper - max(j0, lower + 1)) : 0); }
    __device__ __forceinline__ int next(int j) const { return j < lower ? j + 1 : max(j + 1, upper); }
    __device__ __forceinline__ int first() const { return masked(j0) ? j0 : upper; }
};

// The jobs of all sequences from the longest to the shortest: a sequence of n jobs has one on each of the levels 0 .. n - 1
// (the level-th from its start, so the higher the longer), and they are counted from the highest level down, level by level,
// sequence by sequence. Dealt out in turns that go to and fro over the CTAs, they leave every CTA about the same work
// however the lengths differ. A whole warp looks them up, in ascending order; a lane keeps one of up to 32 sequences. Past
// kLevels sequences every level would cost a look at all of them: then jobs are counted sequence by sequence, which passes
// over the sequences once. Measured, by levels and one by one: one prompt of 16384 rows and 200 of 20 587 - 671 to 767 us by
// their order; 260 of 0-300 67 - 71, 1000 of 0-100 139 - 79, 20000 of one row 24900 - 850.
constexpr int kLevels = 256;
struct Finder {
    const int32_t* cu;
    int B, n_rows, rows, level, before;   // jobs on the levels above, or of the sequences before
    int first;                            // without levels: the sequence of lane 0
    int a, z, n;                          // this lane's sequence, its jobs
    __device__ __forceinline__ void sequence(int s) {
        a = z = 0;
        if (s < B) {
            a = min(max(__ldg(cu + s), 0), n_rows);
            z = min(max(__ldg(cu + s + 1), a), n_rows);
        }
        n = (z - a + rows - 1) / rows;
    }
    __device__ __forceinline__ Finder(const int32_t* cu_, int B_, int n_rows_, int rows_)
        : cu(cu_), B(B_), n_rows(n_rows_), rows(rows_), level(-1), before(0), first(0) {
        const int lane = threadIdx.x & 31;
        if (B > kLevels) {
            sequence(lane);
            return;
        }
        int most = 0;
        for (int s = 0; s < B; s += 32) {
            sequence(s + lane);
            most = max(most, n);
        }
        level = __reduce_max_sync(0xffffffffu, most) - 1;
    }
    __device__ __forceinline__ Job of(int l, int at) const {   // job `at` of lane l's sequence
        const int s0 = __shfl_sync(0xffffffffu, a, l);
        return {s0, __shfl_sync(0xffffffffu, z, l), s0 + at * rows};
    }
    // Job u (not less than the last one); s1 = 0 past the last.
    __device__ __forceinline__ Job find(int u) {
        const int lane = threadIdx.x & 31;
        if (B > kLevels) {
            while (first < B) {
                int up = n;   // jobs up to this lane's
#pragma unroll
                for (int w = 1; w < 32; w <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, up, w);
                    if (lane >= w) up += o;
                }
                const unsigned past = __ballot_sync(0xffffffffu, u - before < up);
                if (past) {
                    const int l = __ffs(past) - 1;
                    return of(l, u - before - __shfl_sync(0xffffffffu, up - n, l));
                }
                before += __shfl_sync(0xffffffffu, up, 31);
                first += 32;
                sequence(first + lane);
            }
            return {0, 0, 0};
        }
        for (; level >= 0; --level) {
            int seen = before;
            for (int s = 0; s < B; s += 32) {
                if (B > 32) sequence(s + lane);
                const unsigned here = __ballot_sync(0xffffffffu, n > level);
                const int rank = u - seen;   // of the ones here
                if (rank < __popc(here)) {
                    const unsigned it = __ballot_sync(0xffffffffu, n > level && __popc(here & ((1u << lane) - 1)) == rank);
                    return of(__ffs(it) - 1, level);
                }
                seen += __popc(here);
            }
            before = seen;
        }
        return {0, 0, 0};
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// tanh(x) of y = 2 log2(e) x: 1 - 2 / (2^y + 1), whose error of 2^-23 is too much of a small x (a large cap); there the series
__device__ __forceinline__ float tanh2(float y) {
    const float x = y * 0.34657359f, x2 = x * x;   // ln(2) / 2
    const float t = fmaf(-2.0f, rcp(ex2(y) + 1.0f), 1.0f), small = x * fmaf(x2, fmaf(x2, 2.0f / 15.0f, -1.0f / 3.0f), 1.0f);
    return fabsf(x) < 0.05f ? small : t;
}
// two f32 operations an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(r)
        : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
          "l"(*reinterpret_cast<unsigned long long*>(&c)));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(r)
        : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&r);
}
// Waits of the roles. Some last as long as a job, which has no bound, so a wait runs out after kTries tries (0.2 s at least) in
// which the CTA made no progress: state[1], which the warp of the products counts up at every key tile, stood still. The most
// that the CTA does between two tiles is to look up a job past a million empty sequences, some 30 ms. A wait that ran out
// marks the CTA (state[0]): every role goes through its loops without waiting, on whatever lies in shared and tensor memory,
// and the CTA ends. Tries and not the clock: its reading at every wait's place cost short prompts 1 us of 23.
constexpr uint32_t kTries = 1u << 24;
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, volatile int* state) {
    int at = -1;
    for (uint32_t n = 1; !mbar_try_wait(bar, parity); ++n) {
        if ((n & 255) != 0) continue;
        if (state[0]) break;
        if (n >= kTries) {
            if (state[1] == at) {
                state[0] = 1;
                break;
            }
            at = state[1];
            n = 0;
        }
    }
}
__device__ __forceinline__ uint32_t ones(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }   // the low n bits
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
template <class E> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// whether either 16-bit float of w has all exponent bits set
template <class E> __device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
    if constexpr (sizeof(E) == 2 && std::is_same<E, __half>::value) return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
    else return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
}

// two values of a type
template <class E> struct Pair;
template <> struct Pair<__half> {
    using type = __half2;
    static __device__ __forceinline__ type of(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
    static __device__ __forceinline__ type zero() { return of(0); }
};
template <> struct Pair<__nv_bfloat16> {
    using type = __nv_bfloat162;
    static __device__ __forceinline__ type of(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
    static __device__ __forceinline__ type zero() { return of(0); }
};

struct Args {
    const int32_t* cu;
    int B, n_rows, HKV, G, R, jobs;   // jobs: as many as there can be
    float c;        // scores to log2 units
    float pre;      // soft cap: 2 log2(e) scale / cap, and c = cap log2(e)
    int window;
    void* out;
    int64_t ldo;
    const void* v;  // for rows that see values which are not finite
    int64_t ldkv;
};

// Adds to the row i of a job, which is written, the values that are not finite and that it sees in the noted rows. Not inlined:
// it hardly ever runs, and its code in the way of the others' costs long prompts 2 %.
template <class E, int D, int BK>
__device__ __noinline__ void add_not_finite(E* out, const E* v, int64_t ldkv, const Job& job, int R, int window, int i, const uint32_t* rows) {
    const Keys<BK> ks(job, R, window);
#pragma unroll 1
    for (int d = 0; d < D; d += 16) {
        float sum[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) sum[e] = 0.0f;
#pragma unroll 1
        for (int j = ks.first(); j < ks.j1; j = ks.next(j))
#pragma unroll 1
            for (int n = 0; n < BK / 32; ++n)
#pragma unroll 1
                for (uint32_t bits = rows[ks.place(j) * (BK / 32) + n]; bits; bits &= bits - 1) {
                    const int k = j * BK + 32 * n + __ffs(bits) - 1;
                    if (k > i || (window > 0 && k <= i - window)) continue;
                    uint4 w[2];
                    const E* x = reinterpret_cast<const E*>(w);
#pragma unroll
                    for (int e = 0; e < 2; ++e) w[e] = reinterpret_cast<const uint4*>(v + k * ldkv + d)[e];
#pragma unroll
                    for (int e = 0; e < 16; ++e) sum[e] += fabsf(to_f32<E>(x[e])) < INFINITY ? 0.0f : to_f32<E>(x[e]);
                }
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (sum[e] != 0.0f) out[d + e] = from_f32<E>(to_f32<E>(out[d + e]) + sum[e]);   // also where it is NaN
    }
}

}  // namespace pk

template <class E, int D, int BK, bool CAP>
__global__ void __launch_bounds__(pk::kThreads, 1)
    k_attention_packed(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const pk::Args A) {
    using namespace pk;
    using namespace tc;
    using M = Smem<D, BK>;
    using Keys = pk::Keys<BK>;
    constexpr int NB = M::NB, NS = M::NS, NH = BK / 64;   // NH: parts in which weights are handed over
    constexpr int B_Q = M::B_Q, B_QFREE = M::B_QFREE, B_FULL = M::B_FULL, B_EMPTY = M::B_EMPTY, B_CLEAN = M::B_CLEAN, B_S = M::B_S,
                  B_P = M::B_P, B_O = M::B_O, B_END = M::B_END, B_DRAIN = M::B_DRAIN, B_JOB = M::B_JOB, B_TAKEN = M::B_TAKEN;
    constexpr bool kBf16 = std::is_same<E, __nv_bfloat16>::value;
    // instruction descriptors: f32 accumulator, A and B of type E, M = 128; B of the second transposed (MN-major)
    constexpr uint32_t kType = (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (8u << 24);
    constexpr uint32_t kDescS = kType | ((uint32_t)(BK / 8) << 17), kDescO = kType | (1u << 16) | ((uint32_t)(D / 8) << 17);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bar = reinterpret_cast<uint64_t*>(sm + M::bar);
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(sm + M::bar + 8 * M::B_COUNT);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);   // and the progress: see wait()
    volatile int* s_odd = s_abort + 2;   // behind the progress: [2 NJ] jobs (counted from 1) in whose masked tiles values that are not finite were met
    volatile int4* s_job = reinterpret_cast<volatile int4*>(s_tmem + 12);   // [NJ] jobs, with the kv head
    uint32_t* s_rows = s_tmem + 12 + 4 * NJ;   // [2 NJ][words] the rows of those, tile after tile
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int R = A.R, G = A.G;
    if (threadIdx.x == kSoft) {
        s_abort[0] = s_abort[1] = 0;
        for (int i = 0; i < 2 * NJ; ++i) s_odd[i] = 0;
        for (int i = 0; i < M::B_COUNT; ++i) {
            mbar_init(&bar[i], i >= B_EMPTY && i < B_CLEAN ? 33 : i >= B_CLEAN && i < B_S ? 32 : i >= B_P && i < B_O ? 128 : i >= B_TAKEN ? 11 : 1);
        }
        mbar_fence_init();
    }
    // tensor memory only after the wait: a kernel that this one follows, and waits for, may still need its own; and a kernel
    // that follows this one may only begin once this one has it: it could take it, and then wait for this one
    pdl_wait();
    if (warp == 8) tmem_alloc(s_tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem = *s_tmem;
    // job n of this CTA, for a whole warp; false past the last
    auto find = [&](int n, Job* job, int* hk) {
        wait(&bar[B_JOB + n % NJ], (uint32_t)(n / NJ) & 1, s_abort);
        const int4 w = {s_job[n % NJ].x, s_job[n % NJ].y, s_job[n % NJ].z, s_job[n % NJ].w};
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[B_TAKEN + n % NJ]);
        *job = {w.x, w.y, w.z};
        *hk = w.w;
        return job->s1 != 0 && !__any_sync(0xffffffffu, *s_abort);
    };
    // ring place i, counted over all jobs; a job of n key tiles takes n + NB: K_0 (and K_1), V_0 with K_NB, .., V_{n-1}
    auto v_at = [&](int i) { return (i % NS) * M::place; };
    auto k_at = [&](int i) { return (i % NS) * M::place + M::tile; };
    auto full = [&](int i) { wait(&bar[B_FULL + i % NS], (uint32_t)((i / NS) & 1), s_abort); };

    if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");   // 256 x 208 + 128 x 88 = 384 x 168
    Job job;
    int hk;
    if (warp == 9) {
        // ---- loads
        int i = 0, loaded = 0;
        for (int q = 0; find(q, &job, &hk); ++q) {
            const Keys ks(job, R, A.window);
            const int tiles = ks.to[1] ? 2 : 1;
            if (lane == 0 && q > 0) wait(&bar[B_QFREE], (uint32_t)((q - 1) & 1), s_abort);
            if (lane == 0 && !*s_abort) {   // a marked CTA brings nothing more
                ++loaded;
                mbar_expect_tx(&bar[B_Q], (uint32_t)(tiles * M::halves * G * R * 128));
                for (int x = 0; x < tiles; ++x)
                    for (int h = 0; h < M::halves; ++h)
                        tma_load_3d(sm + x * M::qtile + h * kHalf, &qmap, 64 * h, hk * G, job.r0 + x * R, &bar[B_Q]);
                for (int j = ks.j0; j < ks.j1 + NB; ++j, ++i) {   // V_{j-NB} and K_j
                    if (i >= NS) wait(&bar[B_EMPTY + i % NS], (uint32_t)((i / NS - 1) & 1), s_abort);
                    if (*s_abort) break;
                    uint64_t* b = &bar[B_FULL + i % NS];
                    mbar_expect_tx(b, (uint32_t)(M::tile * ((j >= ks.j0 + NB) + (j < ks.j1))));
                    for (int h = 0; h < M::halves; ++h) {
                        if (j >= ks.j0 + NB) tma_load_3d(sm + M::ring + v_at(i) + h * M::half, &vmap, 64 * h, hk, job.s0 + (j - NB) * BK, b);
                        if (j < ks.j1) tma_load_3d(sm + M::ring + k_at(i) + h * M::half, &kmap, 64 * h, hk, job.s0 + j * BK, b);
                    }
                }
            }
            __syncwarp();
        }
        if (lane == 0) {
            // copies in flight land before the CTA's shared memory can go
            if (loaded > 0) mbar_wait_bounded(&bar[B_Q], (uint32_t)((loaded - 1) & 1));
            for (int k = i > NS ? i - NS : 0; k < i; ++k) mbar_wait_bounded(&bar[B_FULL + k % NS], (uint32_t)((k / NS) & 1));
        }
        __syncwarp();
    } else if (warp == 8) {
        // ---- products; the warp stays together: uniform operands, one lane issues
        const uint32_t who = elect_one();
        // the K-major descriptor of Q_0, to which the others are steps, and the MN-major one of the first V
        const uint64_t qd = sw128_desc(sm), vd = sw128_mn_desc(sm + M::ring, M::half);
        int i = 0;
        uint32_t clean = 0;            // phases of the places' barriers
        uint32_t given[2] = {0, 0};    // score tiles, over all jobs; they take the places of S_x in turn
        uint32_t seen[2] = {0, 0};     // tiles of weights taken
        auto scores = [&](int x, uint64_t b) {   // S_x = Q_x K^T
            const uint32_t to = given[x]++ % NB;
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                umma_f16_ss(tmem + 128 * x + 64 * to, qd + (uint64_t)((x * M::qtile + (k / 4) * kHalf + (k % 4) * 32) >> 4),
                            b + (uint64_t)(((k / 4) * M::half + (k % 4) * 32) >> 4), kDescS, k > 0, who);
            umma_commit_by(&bar[B_S + 2 * x + to], who);
        };
        for (int q = 0; find(q, &job, &hk); ++q) {
            const Keys ks(job, R, A.window);
            wait(&bar[B_Q], (uint32_t)(q & 1), s_abort);
#pragma unroll 1
            for (int j = ks.j0; j < ks.j0 + NB; ++j) {
                full(i);
                tc_fence_after();
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    if (ks.active(x, j)) scores(x, qd + (uint64_t)((M::ring + k_at(i)) >> 4));
                umma_commit_by(&bar[B_EMPTY + i % NS], who);
                ++i;
            }
            if (ks.j0 + NB >= ks.j1) umma_commit_by(&bar[B_QFREE], who);
            full(i);
            uint32_t fresh[2] = {1, 1};
            for (int j = ks.j0; j < ks.j1; ++j) {   // V_j and K_{j+NB} in place i
                const bool more = j + 1 < ks.j1;
                if (who) s_abort[1] = i;
                if (ks.masked(j)) {
                    const int z = i % NS;
                    wait(&bar[B_CLEAN + z], clean >> z & 1, s_abort);
                    clean ^= 1u << z;
                }
                const uint64_t v = vd + (uint64_t)(v_at(i) >> 4), kn = qd + (uint64_t)((M::ring + k_at(i)) >> 4);
                uint64_t* empty = &bar[B_EMPTY + i % NS];
                ++i;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (ks.active(x, j)) {   // O_x += P_x V_j
                        const uint32_t at = seen[x] % NB;
#pragma unroll
                        for (int h = 0; h < NH; ++h) {   // 64 keys as soon as their weights are there
                            wait(&bar[B_P + 2 * x + at + h], seen[x] / NB & 1, s_abort);
                            tc_fence_after();
#pragma unroll
                            for (int k = 4 * h; k < 4 * h + 4; ++k)
                                umma_f16_ts(tmem + 256 + 128 * x, tmem + 128 * x + 64 * at + 8 * k, v + (uint64_t)(k * 16 * 128 >> 4), kDescO,
                                            !fresh[x] || k > 0, who);
                        }
                        ++seen[x];
                        fresh[x] = 0;
                        if (NB > 1) umma_commit_by(&bar[B_O + x], who);
                        if (j + 1 == ks.to[x]) umma_commit_by(&bar[B_END + x], who);
                    }
                    if (ks.active(x, j + NB)) scores(x, kn);
                    if (more && x == 0) full(i);   // what the next turn reads, looked for while the other tile's weights are formed
                }
                umma_commit_by(empty, who);
                if (j + NB + 1 == ks.j1) umma_commit_by(&bar[B_QFREE], who);   // the job's last scores
            }
        }
        // the MMAs issued so far read shared memory and write tensor memory: they end before either is freed
        umma_commit_by(&bar[B_DRAIN], who);
        mbar_wait_bounded(&bar[B_DRAIN], 0);
        __syncwarp();
    } else if (warp == 11) {
        // ---- what comes next: the others find it in shared memory, instead of each fetching the code that looks it up
        Finder finder(A.cu, A.B, A.n_rows, 2 * R);
        for (int n = 0;; ++n) {
            if (n >= NJ) wait(&bar[B_TAKEN + n % NJ], (uint32_t)(n / NJ - 1) & 1, s_abort);
            const uint32_t id = (uint32_t)n * gridDim.x + (n & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x), unit = id / (uint32_t)A.HKV;
            // lengths that are none (decreasing) may name the same rows over and over: no more jobs than rows can have, and
            // counts that stay far below 2^31
            if (id < (uint32_t)A.jobs) job = finder.find((int)unit);
            else job.s1 = 0;
            if (__any_sync(0xffffffffu, *s_abort)) job.s1 = 0;
            if (lane == 0) {
                s_job[n % NJ].x = job.s0;
                s_job[n % NJ].y = job.s1;
                s_job[n % NJ].z = job.r0;
                s_job[n % NJ].w = (int)(id - unit * A.HKV);
                mbar_arrive(&bar[B_JOB + n % NJ]);
            }
            if (job.s1 == 0) break;
        }
        __syncwarp();
    } else if (warp == 10) {
        // ---- values that are not finite
        int i = 0;
        for (int q = 0; find(q, &job, &hk); ++q) {
            const Keys ks(job, R, A.window);
            uint32_t* rows = s_rows + q % (2 * NJ) * M::words;
            bool marked = false;
            for (int j = ks.j0; j < ks.j1 + NB; ++j, ++i) {   // V_{j-NB} in place i
                // every place in its turn, and released by this warp too: a phase passed over could be taken for another
                full(i);
                if (j >= ks.j0 + NB && ks.masked(j - NB)) {
                    // 0 x each of them, summed: NaN where one is not finite
                    uint4* t = reinterpret_cast<uint4*>(sm + M::ring + v_at(i));
                    typename Pair<E>::type acc[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[k] = Pair<E>::zero();
#pragma unroll 8
                    for (int e = lane; e < M::tile / 16; e += 32) {
                        const uint4 w = t[e];
                        acc[0] = __hfma2(Pair<E>::of(w.x), Pair<E>::zero(), acc[0]);
                        acc[1] = __hfma2(Pair<E>::of(w.y), Pair<E>::zero(), acc[1]);
                        acc[2] = __hfma2(Pair<E>::of(w.z), Pair<E>::zero(), acc[2]);
                        acc[3] = __hfma2(Pair<E>::of(w.w), Pair<E>::zero(), acc[3]);
                    }
                    const auto all = __hadd2(__hadd2(acc[0], acc[1]), __hadd2(acc[2], acc[3]));
                    if (__any_sync(0xffffffffu, !__hbeq2(all, all))) {
                        if (!marked) {
                            if (lane < M::words) rows[lane] = 0;
                            __syncwarp();
                            marked = true;
                        }
                        const int own = job.s1 - job.s0 - (j - NB) * BK;   // rows of the tile that are the sequence's
#pragma unroll 1
                        for (int e = lane; e < M::tile / 16; e += 32) {
                            uint4 w = t[e];
                            uint32_t* u = reinterpret_cast<uint32_t*>(&w);
                            uint32_t some = 0;
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t odd = not_finite2<E>(u[k]);
                                some |= odd;
                                u[k] &= ~((odd >> 15) * 0xFFFFu);
                            }
                            if (!some) continue;
                            t[e] = w;
                            const int r = e / 8 % BK;
                            if (r < own) {
                                atomicOr(rows + ks.place(j - NB) * (BK / 32) + r / 32, 1u << r % 32);
                                s_odd[q % (2 * NJ)] = q + 1;
                            }
                        }
                    }
                    fence_async_smem();
                    mbar_arrive(&bar[B_CLEAN + i % NS]);
                }
                mbar_arrive(&bar[B_EMPTY + i % NS]);
            }
        }
        __syncwarp();
    } else {
        // ---- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int x = warp >> 2, row = threadIdx.x & 127;   // MMA row = tensor-memory lane
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + 128 * x + lanes, to = tmem + 256 + 128 * x + lanes;
        uint32_t n = 0, outs = 0;   // score tiles and outputs taken, over all jobs
        Job next;
        int next_hk;
        bool some = find(0, &next, &next_hk);
        for (int q = 0; some; ++q) {
        job = next;
        hk = next_hk;
        const Keys ks(job, R, A.window);
        const int from = x ? ks.from[1] : ks.from[0], upto = x ? ks.to[1] : ks.to[0];
        const int lo = x ? ks.lo[1] : ks.lo[0], hi = x ? ks.hi[1] : ks.hi[0];
        const int i = lo + row / G;                          // this row's position in the sequence
        const bool live = row < R * G && i <= hi;
        constexpr float kKeep = 1.0f - BK / 16 * kCut;
        float m = -INFINITY, l = 0.0f;
        for (int j = from; j < upto; ++j, ++n) {
            const int kb = j * BK;
            const bool masked = kb + BK - 1 > lo || (A.window > 0 && kb <= hi - A.window);
            const uint32_t at = n % NB, tn = ts + 64 * at;
            wait(&bar[B_S + 2 * x + at], n / NB & 1, s_abort);
            tc_fence_after();
            float s[BK / 32][32];
#pragma unroll
            for (int c = 0; c < BK / 32; ++c) tmem_ld32(tn + 32 * c, s[c]);
            tmem_ld_wait();
            if (CAP) {
#pragma unroll
                for (int c = 0; c < BK / 32; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e) s[c][e] = tanh2(s[c][e] * A.pre);
            }
            if (masked) {
                const int top = i - kb, bottom = A.window > 0 ? top - A.window : -1;   // keys bottom < e <= top are seen
#pragma unroll
                for (int c = 0; c < BK / 32; ++c) {
                    const uint32_t seen = ones(top + 1 - 32 * c) & ~ones(bottom + 1 - 32 * c);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(seen >> e & 1)) s[c][e] = -INFINITY;
                }
            }
            constexpr int C = BK / 16;
            float mm[C];   // chains; a NaN comes through and makes the row's reference NaN
#pragma unroll
            for (int e = 0; e < C; ++e) mm[e] = max3(s[e / 2][16 * (e % 2)], s[e / 2][16 * (e % 2) + 1], s[e / 2][16 * (e % 2) + 2]);
#pragma unroll
            for (int k = 3; k < 15; k += 2)
#pragma unroll
                for (int e = 0; e < C; ++e) mm[e] = max3(mm[e], s[e / 2][16 * (e % 2) + k], s[e / 2][16 * (e % 2) + k + 1]);
#pragma unroll
            for (int e = 0; e < C; e += 2) mm[e] = max3(mm[e], max3(mm[e + 1], s[e / 2][15], s[e / 2][31]), mm[e]);
            const float mx = max3(mm[0], mm[2], C > 4 ? max3(mm[C - 4], mm[C - 2], mm[C - 2]) : mm[0]);
            // not for MMA rows that are nobody's: what lies there (groups that do not divide 128: an earlier kernel's shared memory)
            // may be NaN, and would have the warp rescale at every tile
            const bool raise = live && mx != -INFINITY && !((mx - m) * A.c <= Range<E>::kSlack);   // from -inf, and to NaN, too
            if (__any_sync(0xffffffffu, raise)) {
                const float f = raise ? ex2((m - mx) * A.c) : 1.0f;
                if (raise) m = mx;
                l *= f;
                if (j > from) {
                    if (NB > 1) {   // the product before; the one before that, as with one place the last, ended before these scores
                        wait(&bar[B_O + x], (n - 1) & 1, s_abort);
                        tc_fence_after();
                    }
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        int o[16];
                        uint32_t w[16];
                        tmem_ld16(to + 16 * c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__int_as_float(o[e]) * f);
                        tmem_st16(to + 16 * c, w);
                    }
                }
            }
            const float mc = m == -INFINITY ? 0.0f : __fmaf_rd(-m, A.c, Range<E>::kUp);   // down: no weight passes the bound
            const float2 c2 = make_float2(A.c, A.c), mc2 = make_float2(mc, mc);
            float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
#pragma unroll
            for (int c = 0; c < BK / 32; ++c) {
                uint32_t u[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float2 y = fma2(make_float2(s[c][2 * e], s[c][2 * e + 1]), c2, mc2);
                    y.x = ex2(y.x);
                    y.y = ex2(y.y);
                    if (e & 1) sum1 = add2(sum1, y);
                    else sum0 = add2(sum0, y);
                    u[e] = pack2<E>(y.x, y.y);
                }
                tmem_st16(tn + 16 * c, u);
                if (c % 2) {
                    tmem_st_wait();
                    tc_fence_before();
                    mbar_arrive(&bar[B_P + 2 * x + at + c / 2]);
                }
            }
            sum0 = add2(sum0, sum1);
            l = fmaf(l, kKeep, sum0.x + sum0.y);
        }
        some = find(q + 1, &next, &next_hk);   // while the last products run
        if (!upto) continue;
        wait(&bar[B_END + x], outs & 1, s_abort);
        ++outs;
        tc_fence_after();
        const bool odd = s_odd[q % (2 * NJ)] == q + 1;
        const float inv = *s_abort ? NAN : 1.0f / l;   // nobody takes what a wait that ran out left for an answer
        // 64 columns of the warp's 32 rows at a time by way of shared memory, so that a store instruction writes whole lines
        const uint64_t dst = live ? reinterpret_cast<uint64_t>(static_cast<E*>(A.out) + (int64_t)(job.s0 + i) * A.ldo + (int64_t)(hk * G + row % G) * D) : 0;
        uint8_t* stage = sm + M::out + (threadIdx.x >> 5) * 4096;
#pragma unroll 1   // run once a job: little code rather than many instruction fetches
        for (int c = 0; c < D; c += 64) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (c + 32 * h >= D) break;
                float o[32];
                tmem_ld32(to + c + 32 * h, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= inv;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * h + e) ^ (lane & 7)) << 4)) =
                        make_uint4(pack2<E>(o[8 * e], o[8 * e + 1]), pack2<E>(o[8 * e + 2], o[8 * e + 3]),
                                   pack2<E>(o[8 * e + 4], o[8 * e + 5]), pack2<E>(o[8 * e + 6], o[8 * e + 7]));
            }
            __syncwarp();
#pragma unroll
            for (int r = lane >> 3; r < 32; r += 4) {   // 8 lanes a row
                const uint64_t at = __shfl_sync(0xffffffffu, dst, r);
                const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                if (at && c + 8 * (lane & 7) < D) *reinterpret_cast<uint4*>(at + 2 * c + 16 * (lane & 7)) = w;
            }
            __syncwarp();
        }
        if (odd && live)
            add_not_finite<E, D, BK>(reinterpret_cast<E*>(dst), static_cast<const E*>(A.v) + (int64_t)job.s0 * A.ldkv + (int64_t)hk * D,
                                     A.ldkv, job, A.R, A.window, i, s_rows + q % (2 * NJ) * M::words);
        tc_fence_before();   // O is read before the next job's first weights are handed over
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

namespace {

PFN_cuTensorMapEncodeTiled_v12000 g_encode_packed = nullptr;

bool encode_ready() {
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) == cudaSuccess &&
            r == cudaDriverEntryPointSuccess)
            g_encode_packed = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    });
    return g_encode_packed != nullptr;
}

// rows [n][heads][D] with `ld` values from row to row; boxes of `rows` rows x `heads_box` heads x 64 values
template <class E>
bool make_map(CUtensorMap* m, const void* p, int D, int heads, int n, int64_t ld, int heads_box, int rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)n};
    const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)ld * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)heads_box, (cuuint32_t)rows}, es[3] = {1, 1, 1};
    return g_encode_packed(m, std::is_same<E, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                           3, const_cast<void*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kSMs = 148;
// as many jobs as there can be
int64_t most_jobs(int n_rows, int B, int H, int HKV) {
    return (n_rows / (2 * (128 / (H / HKV))) + std::min<int64_t>(B, n_rows)) * HKV;
}

template <class E, int D, int BK, bool CAP>
cudaError_t launch_packed(const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv, int n_rows,
                          const int32_t* cu, int B, int H, int HKV, float scale, float softcap, int window, void* out,
                          int64_t ldo, cudaStream_t st) {
    using M = pk::Smem<D, BK>;
    const int G = H / HKV, R = 128 / G;
    CUtensorMap qm, km, vm;
    if (!encode_ready()) return cudaErrorNotSupported;
    if (!make_map<E>(&qm, q, D, H, n_rows, ldq, G, R) || !make_map<E>(&km, k, D, HKV, n_rows, ldkv, 1, BK) ||
        !make_map<E>(&vm, v, D, HKV, n_rows, ldkv, 1, BK))
        return cudaErrorInvalidValue;
    static uint64_t set = 0;   // one bit a device; setting it twice does no harm
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!(__atomic_load_n(&set, __ATOMIC_RELAXED) >> (dev & 63) & 1)) {
        e = cudaFuncSetAttribute(k_attention_packed<E, D, BK, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, M::bytes);
        if (e != cudaSuccess) return e;
        __atomic_fetch_or(&set, (uint64_t)1 << (dev & 63), __ATOMIC_RELAXED);
    }
    constexpr float kLog2e = 1.4426950408889634f;
    const int64_t jobs = most_jobs(n_rows, B, H, HKV);
    if (jobs > INT_MAX / 2) return cudaErrorInvalidValue;
    pk::Args a{cu, B, n_rows, HKV, G, R, (int)jobs, CAP ? softcap * kLog2e : scale * kLog2e, CAP ? 2.0f * kLog2e * scale / softcap : 0.0f,
               window, out, ldo, v, ldkv};
    return fbk_launch_early(k_attention_packed<E, D, BK, CAP>, dim3((unsigned)std::min<int64_t>(jobs, kSMs)), dim3(pk::kThreads), (size_t)M::bytes, st, 1, qm,
                      km, vm, a);
}

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" int fbk_attention_packed(int type, const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv,
                                    int n_rows, const int32_t* cu, int B, int H, int HKV, int D, float scale,
                                    float softcap, int window, void* out, int64_t ldo, cudaStream_t st) {
    const bool many = most_jobs(n_rows, B, H, HKV) > kSMs;
#define GO(E, D, BK, CAP) \
    (int)launch_packed<E, D, BK, CAP>(q, ldq, k, v, ldkv, n_rows, cu, B, H, HKV, scale, softcap, window, out, ldo, st)
#define GO_CAP(E, D, BK) (softcap > 0.0f ? GO(E, D, BK, true) : GO(E, D, BK, false))
#define GO_TILE(E, D) (many && n_rows < (int64_t)10 * D * B ? GO_CAP(E, D, 64) : GO_CAP(E, D, 128))
    if (type == T_F16) return D == 128 ? GO_TILE(__half, 128) : D == 96 ? GO_TILE(__half, 96) : GO_TILE(__half, 64);
    return D == 128 ? GO_TILE(__nv_bfloat16, 128) : D == 96 ? GO_TILE(__nv_bfloat16, 96) : GO_TILE(__nv_bfloat16, 64);
#undef GO_TILE
#undef GO_CAP
#undef GO
}
