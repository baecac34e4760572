// attention_packed.cu — causal attention of packed prompts of different lengths.
#include "kv4.cuh"
#include "launch.cuh"

namespace fb {

// CTA = 16 rows of one sequence x one query head; warp w takes the rows
// w, w + 8, .. of the tile, key by key in tiles of 32, lane = key for the
// scores and lane = dimensions l, l + 32, .. for the output.
constexpr int kPkRows = 16, kPkWarps = 8;

// Row range of tile `tile` (of `rows` rows each, the tiles of each sequence
// counted by itself): the sequence's first row and end, and the tile's first
// row; false past the last tile.
__device__ __forceinline__ bool packed_tile(const int32_t* cu, int B, int n_rows, int tile, int rows, int* s0, int* s1,
                                            int* r0) {
    for (int s = 0; s < B; ++s) {
        const int a = min(max(__ldg(cu + s), 0), n_rows), b = min(max(__ldg(cu + s + 1), a), n_rows);
        const int n = (b - a + rows - 1) / rows;
        if (tile < n) {
            *s0 = a;
            *s1 = b;
            *r0 = a + tile * rows;
            return true;
        }
        tile -= n;
    }
    return false;
}

template <class E, int D>
__global__ void __launch_bounds__(32 * kPkWarps) k_attention_packed(const E* __restrict__ q, int64_t ldq,
                                                                    const E* __restrict__ k, const E* __restrict__ v,
                                                                    int64_t ldkv, int n_rows,
                                                                    const int32_t* __restrict__ cu, int B, int H,
                                                                    int HKV, float scale, float softcap, int window,
                                                                    E* out, int64_t ldo) {
    constexpr int NG = D / 32, RW = kPkRows / kPkWarps;
    pdl_trigger();
    pdl_wait();
    int s0, s1, r0;
    if (!packed_tile(cu, B, n_rows, blockIdx.x, kPkRows, &s0, &s1, &r0)) return;
    const int h = blockIdx.y, hk = h / (H / HKV), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ float sk[32][D + 1], sv[32][D], sq[kPkRows][D];
    for (int i = threadIdx.x; i < kPkRows * D; i += blockDim.x) {
        const int r = r0 + i / D;
        sq[i / D][i % D] = r < s1 ? to_f32<E>(q[r * ldq + (int64_t)h * D + i % D]) : 0.0f;
    }
    float m[RW], l[RW], o[RW][NG];
#pragma unroll
    for (int a = 0; a < RW; ++a) {
        m[a] = -INFINITY;
        l[a] = 0.0f;
#pragma unroll
        for (int e = 0; e < NG; ++e) o[a][e] = 0.0f;
    }
    const int last = min(r0 + kPkRows, s1) - 1;
    int j0 = s0;
    if (window > 0) j0 = max(s0, r0 - window + 1);
    for (; j0 <= last; j0 += 32) {
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * D; i += blockDim.x) {
            const int j = j0 + i / D;
            sk[i / D][i % D] = j <= last ? to_f32<E>(k[j * ldkv + (int64_t)hk * D + i % D]) : 0.0f;
            sv[i / D][i % D] = j <= last ? to_f32<E>(v[j * ldkv + (int64_t)hk * D + i % D]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int a = 0; a < RW; ++a) {
            const int r = r0 + warp + a * kPkWarps, j = j0 + lane;
            const bool seen = j <= r && r < s1 && (window <= 0 || j > r - window);
            float s = 0.0f;
            for (int d = 0; d < D; ++d) s = fmaf(sq[warp + a * kPkWarps][d], sk[lane][d], s);
            s *= scale;
            if (softcap > 0.0f) s = softcap * tanhf(s / softcap);
            if (!seen) s = -INFINITY;
            const float mn = fmaxf(m[a], warp_max(s));
            if (!__any_sync(0xffffffffu, seen)) continue;
            const float c = expf(m[a] - mn), p = seen ? expf(s - mn) : 0.0f;
            m[a] = mn;
            l[a] = l[a] * c + warp_sum(p);
#pragma unroll
            for (int e = 0; e < NG; ++e) o[a][e] *= c;
            const unsigned mask = __ballot_sync(0xffffffffu, seen);
            for (int jj = 0; jj < 32; ++jj) {
                const float pj = __shfl_sync(0xffffffffu, p, jj);
                if (!((mask >> jj) & 1)) continue;
#pragma unroll
                for (int e = 0; e < NG; ++e) o[a][e] = fmaf(pj, sv[jj][32 * e + lane], o[a][e]);
            }
        }
    }
#pragma unroll
    for (int a = 0; a < RW; ++a) {
        const int r = r0 + warp + a * kPkWarps;
        if (r >= s1) continue;
#pragma unroll
        for (int e = 0; e < NG; ++e) out[r * ldo + (int64_t)h * D + 32 * e + lane] = from_f32<E>(o[a][e] / l[a]);
    }
}

template <class E, int D>
static cudaError_t launch_packed(const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv, int n_rows,
                                 const int32_t* cu, int B, int H, int HKV, float scale, float softcap, int window,
                                 void* out, int64_t ldo, cudaStream_t st) {
    return fbk_launch(k_attention_packed<E, D>, dim3(n_rows / kPkRows + B, H), dim3(32 * kPkWarps), 0, st, (const E*)q,
                      ldq, (const E*)k, (const E*)v, ldkv, n_rows, cu, B, H, HKV, scale, softcap, window, (E*)out, ldo);
}

}  // namespace fb

using namespace fb;

extern "C" int fbk_attention_packed(int type, const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv,
                                    int n_rows, const int32_t* cu, int B, int H, int HKV, int D, float scale,
                                    float softcap, int window, void* out, int64_t ldo, cudaStream_t st) {
#define GO(E, DD) (int)launch_packed<E, DD>(q, ldq, k, v, ldkv, n_rows, cu, B, H, HKV, scale, softcap, window, out, ldo, st)
    if (type == T_F16) return D == 128 ? GO(__half, 128) : D == 96 ? GO(__half, 96) : GO(__half, 64);
    return D == 128 ? GO(__nv_bfloat16, 128) : D == 96 ? GO(__nv_bfloat16, 96) : GO(__nv_bfloat16, 64);
#undef GO
}
