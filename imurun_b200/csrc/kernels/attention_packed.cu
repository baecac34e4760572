// attention_packed.cu — causal attention of packed prompts of different lengths
// on the 5th-generation tensor cores.
//
//   O_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c s_ij - m_i),  s_ij = q_i . k_j,
// over the keys j that row i sees, c = scale log2(e), m_i a running reference.
//
// A tile is 128 MMA rows: R = 128 / G consecutive rows of one sequence times the
// G query heads of one kv head, so grouped heads share a tile whatever G is and
// short prompts still fill it. A CTA takes two neighbouring tiles (2 R rows),
// which share every key and value tile that it loads. Warps:
//   0..3, 4..7  softmax of tile 0 and 1, a thread a row: scores from tensor
//               memory, mask, row maximum, weights in 16 bits back over the
//               scores' columns; at the end the rows of out;
//   8           the MMAs: S_x = Q_x K_j^T (both from shared memory), then
//               O_x += P_x V_j with P_x from tensor memory. While one tile's
//               warps form weights, the tensor core works for the other:
//               S0 S1 | O0 S0 O1 S1 | O0 S0 O1 S1 ..
//   9           TMA: Q once, then K and V tiles of 128 rows through a ring.
// Tensor memory: S0 S1 (128 columns each, P in their first 64) O0 O1.
//
// The reference m_i is raised only when a tile's maximum exceeds it by 2^8 (the
// weights stay below 256, exact in both types' range), so the accumulator is
// rescaled a few times a row, not once a tile.
#include <cudaTypedefs.h>

#include <mutex>

#include "kv4.cuh"
#include "launch.cuh"
#include "umma.cuh"

namespace fb {
namespace pk {

constexpr int BK = 128, NS = 4;          // keys a tile, ring stages
constexpr int kHalf = 128 * 128;         // 128 rows x 64 values of 16 bits: one SW128 box
constexpr int kSoft = 256, kThreads = kSoft + 64;
constexpr float kRaise = 8.0f;

enum { B_Q = 0, B_FULL = 1, B_EMPTY = B_FULL + NS, B_S = B_EMPTY + NS, B_P = B_S + 2, B_O = B_P + 4, B_DRAIN = B_O + 2,
       B_COUNT = B_DRAIN + 1 };

template <int D>
struct Smem {
    static constexpr int halves = (D + 63) / 64;
    static constexpr int tile = halves * kHalf;            // one Q, K or V tile
    static constexpr int ring = 2 * tile, bar = ring + NS * tile;
    static constexpr int bytes = bar + 8 * B_COUNT + 64 + 1024;
};

struct Job {
    int s0, s1, r0;   // the sequence's rows, the first row of the CTA's tiles
};

// The CTA's tile: sequences in order, each from its last (longest) tile to its
// first; 32 sequences at a time, one a lane. s1 = 0 past the last tile.
__device__ __forceinline__ Job find_job(const int32_t* cu, int B, int n_rows, int tile, int rows) {
    const int lane = threadIdx.x & 31;
    for (int b = 0; b < B; b += 32) {
        int a = 0, z = 0;
        if (b + lane < B) {
            a = min(max(__ldg(cu + b + lane), 0), n_rows);
            z = min(max(__ldg(cu + b + lane + 1), a), n_rows);
        }
        const int n = (z - a + rows - 1) / rows;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, sum > tile);
        if (past) {
            const int l = __ffs(past) - 1;
            const int r = a + (sum - 1 - tile) * rows;   // lane l: tile - (sum - n) counted from its end
            return {__shfl_sync(0xffffffffu, a, l), __shfl_sync(0xffffffffu, z, l), __shfl_sync(0xffffffffu, r, l)};
        }
        tile -= __shfl_sync(0xffffffffu, sum, 31);
    }
    return {0, 0, 0};
}

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

struct Args {
    const int32_t* cu;
    int B, n_rows, HKV, G, R;
    float c;        // scores to log2 units
    float pre;      // soft cap: 2 log2(e) scale / cap, and c = cap log2(e)
    int window;
    void* out;
    int64_t ldo;
    const void* v;  // for rows that see values which are not finite
    int64_t ldkv;
};

}  // namespace pk

template <class E, int D, bool CAP>
__global__ void __launch_bounds__(pk::kThreads, 1)
    k_attention_packed(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const pk::Args A) {
    using namespace pk;
    using namespace tc;
    using M = Smem<D>;
    constexpr bool kBf16 = std::is_same<E, __nv_bfloat16>::value;
    // instruction descriptors: f32 accumulator, A and B of type E, M = 128; B of the second transposed (MN-major)
    constexpr uint32_t kType = (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (8u << 24);
    constexpr uint32_t kDescS = kType | ((uint32_t)(BK / 8) << 17), kDescO = kType | (1u << 16) | ((uint32_t)(D / 8) << 17);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bar = reinterpret_cast<uint64_t*>(sm + M::bar);
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(sm + M::bar + 8 * B_COUNT);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
    volatile int* s_odd = s_abort + 1;                       // values that are not finite were met
    Job* s_job = reinterpret_cast<Job*>(s_tmem + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hk = blockIdx.x % A.HKV, R = A.R, G = A.G;
    pdl_trigger();
    pdl_wait();
    if (warp == 0) {
        const Job j = find_job(A.cu, A.B, A.n_rows, blockIdx.x / A.HKV, 2 * R);
        if (lane == 0) *s_job = j;
    }
    if (threadIdx.x == kSoft) {
        *s_abort = 0;
        *s_odd = 0;
        mbar_init(&bar[B_Q], 1);
        for (int s = 0; s < NS; ++s) {
            mbar_init(&bar[B_FULL + s], 1);
            mbar_init(&bar[B_EMPTY + s], 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&bar[B_S + x], 1);
            mbar_init(&bar[B_P + 2 * x], 128);
            mbar_init(&bar[B_P + 2 * x + 1], 128);
            mbar_init(&bar[B_O + x], 1);
        }
        mbar_init(&bar[B_DRAIN], 1);
        mbar_fence_init();
    }
    __syncthreads();
    const int s0 = s_job->s0, s1 = s_job->s1, r0 = s_job->r0;
    if (s1 == 0) return;
    if (warp == 8) tmem_alloc(s_tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    // key tiles [first[x], end[x]) of tile x, counted from the sequence's start
    int first[2], end[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int lo = r0 + x * R - s0, hi = min(lo + R, s1 - s0) - 1;   // rows of the tile
        first[x] = A.window > 0 ? max(0, lo - A.window + 1) / BK : 0;
        end[x] = lo < s1 - s0 ? hi / BK + 1 : 0;
    }
    const int j0 = first[0], j1 = max(end[0], end[1]);
    const int tiles = end[1] ? 2 : 1;

    if (warp == 9) {
        if (lane == 0) {
            mbar_expect_tx(&bar[B_Q], (uint32_t)(tiles * M::halves * G * R * 128));
            for (int x = 0; x < tiles; ++x)
                for (int h = 0; h < M::halves; ++h)
                    tma_load_3d(sm + x * M::tile + h * kHalf, &qmap, 64 * h, hk * G, r0 + x * R, &bar[B_Q]);
            int i = 0;
            const int n = 2 * (j1 - j0);   // K and V tiles in turn
            for (; i < n; ++i) {
                const int st = i % NS;
                if (i >= NS && !mbar_wait(&bar[B_EMPTY + st], (uint32_t)((i / NS - 1) & 1), s_abort)) break;
                mbar_expect_tx(&bar[B_FULL + st], (uint32_t)M::tile);
                for (int h = 0; h < M::halves; ++h)
                    tma_load_3d(sm + M::ring + st * M::tile + h * kHalf, i & 1 ? &vmap : &kmap, 64 * h, hk,
                                s0 + (j0 + i / 2) * BK, &bar[B_FULL + st]);
            }
            if (i < n) *s_abort = 1;
            // copies in flight land before the CTA's shared memory can go
            mbar_wait_bounded(&bar[B_Q], 0);
            for (int k = i > NS ? i - NS : 0; k < i; ++k) mbar_wait_bounded(&bar[B_FULL + k % NS], (uint32_t)((k / NS) & 1));
        }
    } else if (warp == 8) {
        if (lane == 0) {
            const uint64_t q0 = sw128_desc(sm), k0 = sw128_desc(sm + M::ring);
            const uint64_t v0 = sw128_mn_desc(sm + M::ring, kHalf);
            auto stage = [&](int i) { return (uint64_t)((i % NS) * M::tile >> 4); };
            auto full = [&](int i) {
                const bool ok = mbar_wait(&bar[B_FULL + i % NS], (uint32_t)((i / NS) & 1), s_abort);
                tc_fence_after();
                return ok;
            };
            auto scores = [&](int x, int j) {   // S_x = Q_x K_j^T
                const uint64_t a = q0 + (uint64_t)(x * M::tile >> 4), b = k0 + stage(2 * (j - j0));
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint64_t o = (uint64_t)(((k / 4) * kHalf + (k % 4) * 32) >> 4);
                    umma_f16_ss(tmem + 128 * x, a + o, b + o, kDescS, k > 0);
                }
                umma_commit(&bar[B_S + x]);
            };
            auto active = [&](int x, int j) { return j >= first[x] && j < end[x]; };
            int n[2] = {0, 0};   // weight tiles taken
            bool ok = mbar_wait(&bar[B_Q], 0, s_abort) && full(0);
            if (ok) {
                for (int x = 0; x < 2; ++x)
                    if (active(x, j0)) scores(x, j0);
                umma_commit(&bar[B_EMPTY + 0]);
            }
            for (int j = j0; j < j1 && ok; ++j) {
                const bool more = j + 1 < j1;
                const int iv = 2 * (j - j0) + 1;
                if (more) ok = full(iv + 1);
                ok = ok && full(iv);
                for (int x = 0; x < 2 && ok; ++x) {
                    if (active(x, j)) {
                        const uint64_t b = v0 + stage(iv);
                        for (int h = 0; h < 2 && ok; ++h) {   // 64 keys as soon as their weights are there
                            ok = mbar_wait(&bar[B_P + 2 * x + h], (uint32_t)(n[x] & 1), s_abort);
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll
                            for (int k = 4 * h; k < 4 * h + 4; ++k)
                                umma_f16_ts(tmem + 256 + 128 * x, tmem + 128 * x + 8 * k, b + (uint64_t)(k * 16 * 128 >> 4), kDescO,
                                            n[x] > 0 || k > 0);
                        }
                        if (!ok) break;
                        ++n[x];
                        if (j + 1 == end[x]) umma_commit(&bar[B_O + x]);
                    }
                    if (more && active(x, j + 1)) scores(x, j + 1);
                }
                if (!ok) break;
                umma_commit(&bar[B_EMPTY + iv % NS]);
                if (more) umma_commit(&bar[B_EMPTY + (iv + 1) % NS]);
            }
            if (!ok) *s_abort = 1;
            umma_commit(&bar[B_DRAIN]);
            mbar_wait_bounded(&bar[B_DRAIN], 0);
        }
        __syncwarp();
    } else {
        const int x = warp >> 2, row = threadIdx.x & 127;   // MMA row = tensor-memory lane
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + 128 * x + lanes, to = tmem + 256 + 128 * x + lanes;
        const int lo = r0 + x * R - s0, hi = min(lo + R, s1 - s0) - 1;
        const int i = lo + row / G;                          // this row's position in the sequence
        const bool live = row < R * G && i <= hi;
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = first[x]; j < end[x]; ++j) {
            const int kb = j * BK;
            const bool masked = kb + BK - 1 > lo || (A.window > 0 && kb <= hi - A.window);
            if (masked) {
                // values that a row does not see must not reach it as 0 x inf: the tile's
                // values that are not finite become 0, and the rows that see them get them at the end
                const int iv = 2 * (j - j0) + 1;
                ok = mbar_wait(&bar[B_FULL + iv % NS], (uint32_t)((iv / NS) & 1), s_abort);
                if (!ok) break;
                uint4* t = reinterpret_cast<uint4*>(sm + M::ring + (iv % NS) * M::tile);
                bool odd = false;
                for (int e = row; e < M::tile / 16; e += 128) {
                    uint4 w = t[e];
                    if (not_finite2<E>(w.x) | not_finite2<E>(w.y) | not_finite2<E>(w.z) | not_finite2<E>(w.w)) {
                        uint32_t* u = reinterpret_cast<uint32_t*>(&w);
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t b = not_finite2<E>(u[k]);
                            u[k] &= ~((b >> 15) * 0xFFFFu);
                        }
                        t[e] = w;
                        odd = true;
                    }
                }
                if (odd) *s_odd = 1;
                fence_async_smem();
            }
            ok = mbar_wait(&bar[B_S + x], (uint32_t)((j - first[x]) & 1), s_abort);
            if (!ok) break;
            tc_fence_after();
            float s[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, s[c]);
            tmem_ld_wait();
            if (CAP) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e) s[c][e] = fmaf(-2.0f, rcp(ex2(s[c][e] * A.pre) + 1.0f), 1.0f);   // tanh
            }
            if (masked) {
                const int top = i - kb, bottom = A.window > 0 ? top - A.window : -1;   // keys bottom < e <= top are seen
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * c + e > top || 32 * c + e <= bottom) s[c][e] = -INFINITY;
            }
            float mm[8];   // eight chains of three-operand maxima
#pragma unroll
            for (int e = 0; e < 8; ++e) mm[e] = fmaxf(s[e / 2][16 * (e % 2)], s[e / 2][16 * (e % 2) + 1]);
#pragma unroll
            for (int u = 2; u < 16; u += 2)
#pragma unroll
                for (int e = 0; e < 8; ++e) mm[e] = fmaxf(fmaxf(mm[e], s[e / 2][16 * (e % 2) + u]), s[e / 2][16 * (e % 2) + u + 1]);
            const float mx = fmaxf(fmaxf(fmaxf(mm[0], mm[1]), fmaxf(mm[2], mm[3])), fmaxf(fmaxf(mm[4], mm[5]), fmaxf(mm[6], mm[7])));
            if (j == first[x]) {
                m = mx;
            } else {
                const bool raise = (mx - m) * A.c > kRaise;   // also from -inf
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = raise ? ex2((m - mx) * A.c) : 1.0f;
                    if (raise) m = mx;
                    l *= f;
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        int o[16];
                        uint32_t u[16];
                        tmem_ld16(to + 16 * c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(__int_as_float(o[e]) * f);
                        tmem_st16(to + 16 * c, u);
                    }
                }
            }
            const float2 c2 = make_float2(A.c, A.c), mc2 = m == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(-m * A.c, -m * A.c);
            float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t u[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float2 y = fma2(make_float2(s[2 * h + e / 16][2 * e % 32], s[2 * h + e / 16][2 * e % 32 + 1]), c2, mc2);
                    y.x = ex2(y.x);
                    y.y = ex2(y.y);
                    if (e & 1) sum1 = add2(sum1, y);
                    else sum0 = add2(sum0, y);
                    u[e] = pack2<E>(y.x, y.y);
                }
                tmem_st32(ts + 32 * h, u);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&bar[B_P + 2 * x + h]);
            }
            sum0 = add2(sum0, sum1);
            l += sum0.x + sum0.y;
        }
        if (ok && end[x]) {
            ok = mbar_wait(&bar[B_O + x], 0, s_abort);
            tc_fence_after();
        }
        if (!ok) *s_abort = 1;
        asm volatile("bar.sync 1, 256;" ::: "memory");       // both tiles' finds
        const bool odd = *s_odd != 0;
        if (ok && end[x]) {
            const float inv = 1.0f / l;
            E* dst = static_cast<E*>(A.out) + (int64_t)(s0 + i) * A.ldo + (int64_t)(hk * G + row % G) * D;
            const E* v = static_cast<const E*>(A.v) + (int64_t)s0 * A.ldkv + (int64_t)hk * D;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                float o[32];
                tmem_ld32(to + 32 * c, o);
                tmem_ld_wait();
                if (live) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] *= inv;
                    if (odd) {
                        for (int k = A.window > 0 ? max(0, i - A.window + 1) : 0; k <= i; ++k)
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float y = to_f32<E>(v[k * A.ldkv + 32 * c + e]);
                                if (!(fabsf(y) < INFINITY)) o[e] += y;
                            }
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        *reinterpret_cast<uint4*>(dst + 32 * c + e) =
                            make_uint4(pack2<E>(o[e], o[e + 1]), pack2<E>(o[e + 2], o[e + 3]), pack2<E>(o[e + 4], o[e + 5]),
                                       pack2<E>(o[e + 6], o[e + 7]));
                }
            }
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

template <class E, int D, bool CAP>
cudaError_t launch_packed(const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv, int n_rows,
                          const int32_t* cu, int B, int H, int HKV, float scale, float softcap, int window, void* out,
                          int64_t ldo, cudaStream_t st) {
    using M = pk::Smem<D>;
    const int G = H / HKV, R = 128 / G;
    CUtensorMap qm, km, vm;
    if (!encode_ready()) return cudaErrorNotSupported;
    if (!make_map<E>(&qm, q, D, H, n_rows, ldq, G, R) || !make_map<E>(&km, k, D, HKV, n_rows, ldkv, 1, pk::BK) ||
        !make_map<E>(&vm, v, D, HKV, n_rows, ldkv, 1, pk::BK))
        return cudaErrorInvalidValue;
    static uint64_t set = 0;   // one bit a device; setting it twice does no harm
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!(__atomic_load_n(&set, __ATOMIC_RELAXED) >> (dev & 63) & 1)) {
        e = cudaFuncSetAttribute(k_attention_packed<E, D, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, M::bytes);
        if (e != cudaSuccess) return e;
        __atomic_fetch_or(&set, (uint64_t)1 << (dev & 63), __ATOMIC_RELAXED);
    }
    constexpr float kLog2e = 1.4426950408889634f;
    pk::Args a{cu, B, n_rows, HKV, G, R, CAP ? softcap * kLog2e : scale * kLog2e, CAP ? 2.0f * kLog2e * scale / softcap : 0.0f,
               window, out, ldo, v, ldkv};
    const int64_t tiles = n_rows / (2 * R) + std::min<int64_t>(B, n_rows);
    return fbk_launch_early(k_attention_packed<E, D, CAP>, dim3((unsigned)(tiles * HKV)), dim3(pk::kThreads), (size_t)M::bytes, st, qm,
                      km, vm, a);
}

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" int fbk_attention_packed(int type, const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv,
                                    int n_rows, const int32_t* cu, int B, int H, int HKV, int D, float scale,
                                    float softcap, int window, void* out, int64_t ldo, cudaStream_t st) {
#define GO(E, DD)                                                                                                           \
    (int)(softcap > 0.0f                                                                                                    \
              ? launch_packed<E, DD, true>(q, ldq, k, v, ldkv, n_rows, cu, B, H, HKV, scale, softcap, window, out, ldo, st) \
              : launch_packed<E, DD, false>(q, ldq, k, v, ldkv, n_rows, cu, B, H, HKV, scale, softcap, window, out, ldo, st))
    if (type == T_F16) return D == 128 ? GO(__half, 128) : D == 96 ? GO(__half, 96) : GO(__half, 64);
    return D == 128 ? GO(__nv_bfloat16, 128) : D == 96 ? GO(__nv_bfloat16, 96) : GO(__nv_bfloat16, 64);
#undef GO
}
