// kv4.cu — the paged cache held in 4 bits: append with RoPE, and attention of
// single tokens over it.
#include "kv4.cuh"
#include "launch.cuh"

namespace fb {

// ================================================================ append
// CTA y of token x takes the heads hpc y .. hpc (y + 1) - 1 of the token's
// H + 2 HKV (q, then k, then v); a thread owns 8 consecutive dimensions (one
// 16-byte load of 16-bit values) and walks over the heads, so the token's
// cos and sin stay in registers. A group of 32 values is four neighbouring
// threads: its extremes by two shuffles, its codes one 32-bit word of K or
// two 16-bit words of V a thread. Rotation and quantisation are in 32 bits
// with every step rounded by itself (no fused multiply-add), so the codes are
// those of the plain formula.
template <class E, class O, int D>
__global__ void __launch_bounds__(256) k_kv4_append(const __grid_constant__ fbx_kv4_cache c, const E* q, const E* k,
                                                    const E* v, int64_t ldq, int64_t ldkv, int H, int hpc,
                                                    const int32_t* __restrict__ tok_seq,
                                                    const int32_t* __restrict__ tok_pos, int rot, int neox,
                                                    const float* __restrict__ rcos, const float* __restrict__ rsin,
                                                    int n_rope, O* q_out, int64_t ldq_out, O* k_out, O* v_out,
                                                    int64_t ldkv_out) {
    using R = Kv4Rec<D>;
    constexpr int L = D / 8;   // threads a head
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, HKV = c.n_head_kv;
    const int pos = tok_pos[t];
    if (pos < 0) return;   // padding
    const int seq = tok_seq[t];
    if (seq < 0 || seq >= c.n_seqs || pos >= n_rope) {
        if (c.err && threadIdx.x == 0) atomicExch(c.err, 6);
        return;
    }
    const int page = kv4_page(c, seq, pos / kKv4Page), row = pos % kKv4Page;
    if (page < 0) return;
    const int d0 = (threadIdx.x % L) * 8, half = rot / 2;
    // cos and sin of this thread's 8 dimensions, and where their partners are
    float cs[8], sn[8];
    int other[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        cs[i] = 1.0f;
        sn[i] = 0.0f;
        other[i] = d;
        if (d < rot) {
            const int pair = neox ? (d < half ? d : d - half) : d / 2;
            const bool first = neox ? d < half : d % 2 == 0;
            cs[i] = __ldg(rcos + (size_t)pos * half + pair);
            sn[i] = __ldg(rsin + (size_t)pos * half + pair);
            if (first) sn[i] = -sn[i];   // x0 cos - x1 sin, and x1 cos + x0 sin for the second
            other[i] = neox ? (first ? d + half : d - half) : d ^ 1;
        }
    }
    const int h1 = min(hpc * ((int)blockIdx.y + 1), H + 2 * HKV), step = blockDim.x / L;
    // whole warps walk together (the shuffles below): a head past the end repeats nothing but takes part
    for (int hb = hpc * blockIdx.y; hb < h1; hb += step) {
        const int h = hb + threadIdx.x / L;
        const bool live = h < h1;
        const int kind = !live ? 3 : h < H ? 0 : h < H + HKV ? 1 : 2;
        const int hk = kind == 1 ? h - H : kind == 2 ? h - H - HKV : 0;
        const E* src = kind == 0 ? q + t * ldq + h * D : kind == 1 ? k + t * ldkv + hk * D : v + t * ldkv + hk * D;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
        if (live) load8(src + d0, x);
        if (kind < 2 && d0 < rot) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float o = to_f32<E>(src[other[i]]);
                y[i] = d0 + i < rot ? __fadd_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(o, sn[i])) : x[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = y[i];
        }
        // every read of the head before any write: the outputs may be the inputs
        if constexpr (32 % L == 0) __syncwarp();
        else __syncthreads();
        float lo = INFINITY, hi = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
        }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        if (kind == 0) {
            store8(q_out + t * ldq_out + h * D + d0, x);
        } else if (live) {
            if (!(lo <= hi)) lo = hi = 0.0f;   // nothing but NaN
            const __half lo16 = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
            lo = __half2float(lo16);
            const __half d16 = __float2half_rn(__fmul_rn(__fsub_rn(fminf(fmaxf(hi, -65504.0f), 65504.0f), lo), 1.0f / 15.0f));
            const float d = __half2float(d16), inv = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float code = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], lo), inv)), 0.0f), 15.0f);
                word |= (uint32_t)code << (4 * i);
                x[i] = __fadd_rn(lo, __fmul_rn(d, code));
            }
            uint8_t* rec = kv4_record(c, page, hk, R::bytes);
            const int g = d0 / 32, u = (d0 / 8) % 4;
            if (kind == 1) {
                *reinterpret_cast<uint32_t*>(rec + row * R::row + 4 * R::NG * u + 4 * g) = word;
            } else {
                const int turn = ((row >> 1) & 1) * 4;
                uint8_t* at = rec + R::v + row * R::row + 2 * g;
                *reinterpret_cast<uint16_t*>(at + 2 * R::NG * ((2 * u) ^ turn)) = (uint16_t)word;
                *reinterpret_cast<uint16_t*>(at + 2 * R::NG * ((2 * u + 1) ^ turn)) = (uint16_t)(word >> 16);
            }
            if (u == 0) {
                __half* sc = reinterpret_cast<__half*>(rec + (kind == 1 ? R::kd : R::vd)) + row * R::GP + g;
                sc[0] = d16;
                sc[kKv4Page * R::GP] = lo16;
            }
            O* told = kind == 1 ? k_out : v_out;
            if (told) store8(told + t * ldkv_out + hk * D + d0, x);
        }
    }
}

// ================================================================ attention
// One CTA a (token, kv head, 8 of its query heads); warp w takes the pages
// w, w + 8, .. of the token's context, lane l the dimensions l, l + 32, ..
constexpr int kV1Warps = 8;

__device__ __forceinline__ float code_at(const uint8_t* row, int byte, int n) { return (float)((row[byte] >> (4 * (n & 1))) & 15); }

template <class E, int D>
__global__ void __launch_bounds__(32 * kV1Warps) k_kv4_attention(const __grid_constant__ fbx_kv4_cache c,
                                                                 const E* __restrict__ q, int64_t ldq, int H,
                                                                 const int32_t* __restrict__ tok_seq,
                                                                 const int32_t* __restrict__ tok_pos, float scale,
                                                                 float softcap, int window, E* out, int64_t ldo) {
    using R = Kv4Rec<D>;
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.z, hk = blockIdx.y, G = H / c.n_head_kv, g0 = blockIdx.x * 8, gn = min(8, G - g0);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pos = tok_pos[t];
    if (pos < 0) return;
    const int seq = tok_seq[t];
    const bool known = seq >= 0 && seq < c.n_seqs;
    if (!known && c.err && threadIdx.x == 0) atomicExch(c.err, 6);
    __shared__ float sq[8][D], sm[kV1Warps][8], sl[kV1Warps][8], so[kV1Warps][8][D];
    for (int i = threadIdx.x; i < 8 * D; i += blockDim.x)
        sq[i / D][i % D] = i / D < gn ? to_f32<E>(q[t * ldq + (int64_t)(hk * G + g0 + i / D) * D + i % D]) : 0.0f;
    __syncthreads();
    float m[8], l[8], o[8][R::NG];
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
#pragma unroll
        for (int e = 0; e < R::NG; ++e) o[g][e] = 0.0f;
    }
    const int first = window > 0 ? max(0, pos - window + 1) : 0;
    for (int i = first / kKv4Page + warp; known && i <= pos / kKv4Page; i += kV1Warps) {
        const int page = kv4_page(c, seq, i);
        if (page < 0) continue;
        const uint8_t* rec = kv4_record(c, page, hk, R::bytes);
        for (int j = 0; j < kKv4Page; ++j) {
            const int key = i * kKv4Page + j;
            if (key < first || key > pos) continue;
            const int n = lane % 8, u = lane / 8, h = lane / 4;
            float kx[R::NG], vx[R::NG];
#pragma unroll
            for (int e = 0; e < R::NG; ++e) {
                const __half* sk = reinterpret_cast<const __half*>(rec + R::kd) + j * R::GP + e;
                const __half* sv = reinterpret_cast<const __half*>(rec + R::vd) + j * R::GP + e;
                kx[e] = __half2float(sk[kKv4Page * R::GP]) +
                        __half2float(sk[0]) * code_at(rec + j * R::row, 4 * R::NG * u + 4 * e + n / 2, n);
                const int hh = h ^ (((j >> 1) & 1) * 4);
                vx[e] = __half2float(sv[kKv4Page * R::GP]) +
                        __half2float(sv[0]) * code_at(rec + R::v + j * R::row, 2 * R::NG * hh + 2 * e + (lane % 4) / 2, lane);
            }
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                if (g >= gn) break;
                float s = 0.0f;
#pragma unroll
                for (int e = 0; e < R::NG; ++e) s += sq[g][32 * e + lane] * kx[e];
                s = warp_sum(s) * scale;
                if (softcap > 0.0f) s = softcap * tanhf(s / softcap);
                const float mn = fmaxf(m[g], s), a = expf(m[g] - mn), p = expf(s - mn);
                m[g] = mn;
                l[g] = l[g] * a + p;
#pragma unroll
                for (int e = 0; e < R::NG; ++e) o[g][e] = o[g][e] * a + p * vx[e];
            }
        }
    }
    for (int g = 0; g < gn; ++g) {
        if (lane == 0) {
            sm[warp][g] = m[g];
            sl[warp][g] = l[g];
        }
        for (int e = 0; e < R::NG; ++e) so[warp][g][32 * e + lane] = o[g][e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < gn * D; i += blockDim.x) {
        const int g = i / D, d = i % D;
        float M = -INFINITY, S = 0.0f, O = 0.0f;
        for (int w = 0; w < kV1Warps; ++w) M = fmaxf(M, sm[w][g]);
        for (int w = 0; w < kV1Warps; ++w) {
            if (sm[w][g] == -INFINITY) continue;
            const float a = expf(sm[w][g] - M);
            S += sl[w][g] * a;
            O += so[w][g][d] * a;
        }
        out[t * ldo + (int64_t)(hk * G + g0 + g) * D + d] = from_f32<E>(S > 0.0f ? O / S : 0.0f);
    }
}

// ---------------------------------------------------------------- launches

struct AppendArgs {
    fbx_kv4_cache c;
    const void *q, *k, *v;
    int64_t ldq, ldkv;
    int T, H;
    const int32_t *tok_seq, *tok_pos;
    int rot, neox;
    const float *rcos, *rsin;
    int n_rope;
    void* q_out;
    int64_t ldq_out;
    void *k_out, *v_out;
    int64_t ldkv_out;
};

template <class E, class O, int D>
static cudaError_t launch_append(const AppendArgs& a, cudaStream_t st) {
    const int H = a.q ? a.H : 0, heads = H + 2 * a.c.n_head_kv;
    const int threads = D == 96 ? 192 : 256, per = threads / (D / 8);
    // few tokens: a CTA a run of heads; many: a token's heads in one CTA
    const int hpc = a.T >= 148 ? heads : per;
    return fbk_launch(k_kv4_append<E, O, D>, dim3(a.T, (heads + hpc - 1) / hpc), dim3(threads), 0, st, a.c,
                      (const E*)a.q, (const E*)a.k, (const E*)a.v, a.ldq, a.ldkv, H, hpc, a.tok_seq, a.tok_pos, a.rot,
                      a.neox, a.rcos, a.rsin, a.n_rope, (O*)a.q_out, a.ldq_out, (O*)a.k_out, (O*)a.v_out, a.ldkv_out);
}
template <class E, class O>
static cudaError_t append_d(const AppendArgs& a, cudaStream_t st) {
    return a.c.head_dim == 128 ? launch_append<E, O, 128>(a, st)
         : a.c.head_dim == 96 ? launch_append<E, O, 96>(a, st) : launch_append<E, O, 64>(a, st);
}
template <class E>
static cudaError_t append_o(const AppendArgs& a, int out_type, cudaStream_t st) {
    return out_type == T_F32 ? append_d<E, float>(a, st)
         : out_type == T_F16 ? append_d<E, __half>(a, st) : append_d<E, __nv_bfloat16>(a, st);
}

template <class E, int D>
static cudaError_t launch_kv4_attention(const fbx_kv4_cache& c, const void* q, int64_t ldq, int T, int H,
                                        const int32_t* tok_seq, const int32_t* tok_pos, float scale, float softcap,
                                        int window, void* out, int64_t ldo, cudaStream_t st) {
    const int G = H / c.n_head_kv;
    return fbk_launch(k_kv4_attention<E, D>, dim3((G + 7) / 8, c.n_head_kv, T), dim3(32 * kV1Warps), 0, st, c,
                      (const E*)q, ldq, H, tok_seq, tok_pos, scale, softcap, window, (E*)out, ldo);
}
template <class E>
static cudaError_t kv4_attention_d(const fbx_kv4_cache& c, const void* q, int64_t ldq, int T, int H,
                                   const int32_t* tok_seq, const int32_t* tok_pos, float scale, float softcap,
                                   int window, void* out, int64_t ldo, cudaStream_t st) {
    return c.head_dim == 128 ? launch_kv4_attention<E, 128>(c, q, ldq, T, H, tok_seq, tok_pos, scale, softcap, window, out, ldo, st)
         : c.head_dim == 96 ? launch_kv4_attention<E, 96>(c, q, ldq, T, H, tok_seq, tok_pos, scale, softcap, window, out, ldo, st)
                            : launch_kv4_attention<E, 64>(c, q, ldq, T, H, tok_seq, tok_pos, scale, softcap, window, out, ldo, st);
}

}  // namespace fb

using namespace fb;

extern "C" int fbk_kv4_append(const fbx_kv4_cache& c, int type, const void* q, const void* k, const void* v, int64_t ldq,
                              int64_t ldkv, int T, int H, const int32_t* tok_seq, const int32_t* tok_pos, int rot, int neox,
                              const float* rcos, const float* rsin, int n_rope, int out_type, void* q_out, int64_t ldq_out,
                              void* k_out, void* v_out, int64_t ldkv_out, cudaStream_t st) {
    const AppendArgs a{c, q, k, v, ldq, ldkv, T, H, tok_seq, tok_pos, rot, neox, rcos, rsin, n_rope, q_out, ldq_out,
                       k_out, v_out, ldkv_out};
    return (int)(type == T_F32 ? append_o<float>(a, out_type, st)
               : type == T_F16 ? append_o<__half>(a, out_type, st) : append_o<__nv_bfloat16>(a, out_type, st));
}

extern "C" size_t fbk_kv4_attention_workspace(int, int, int, int, int) { return 0; }

extern "C" int fbk_kv4_attention(const fbx_kv4_cache& c, int type, const void* q, int64_t ldq, int T, int H,
                                 const int32_t* tok_seq, const int32_t* tok_pos, int, float scale, float softcap,
                                 int window, void* out, int64_t ldo, void*, cudaStream_t st) {
    return (int)(type == T_F32 ? kv4_attention_d<float>(c, q, ldq, T, H, tok_seq, tok_pos, scale, softcap, window, out, ldo, st)
               : type == T_F16 ? kv4_attention_d<__half>(c, q, ldq, T, H, tok_seq, tok_pos, scale, softcap, window, out, ldo, st)
                               : kv4_attention_d<__nv_bfloat16>(c, q, ldq, T, H, tok_seq, tok_pos, scale, softcap, window, out, ldo, st));
}
