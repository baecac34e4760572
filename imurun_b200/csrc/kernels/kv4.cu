// kv4.cu — the paged cache held in 4 bits: append with RoPE, and attention of
// single tokens over it.
#include <cooperative_groups.h>

#include <algorithm>

#include "kv4.cuh"
#include "launch.cuh"
#include "tma.cuh"

namespace fb {

// ================================================================ append
// CTA y of token x takes the heads hpc y .. hpc (y + 1) - 1 of the token's
// H + 2 HKV (q, then k, then v), a warp 32 / (D / 8) heads at a time, a lane 8
// consecutive dimensions (one 16-byte load of 16-bit values). What bounds it is
// memory: a lane's loads of U heads are issued before anything else, under the
// chain of position, page and rotation that the stores wait for, and the cos and
// sin of its 8 dimensions serve all its heads. Where a lane's 8 dimensions are
// rotated together or not at all, the partner of a value is in the same lane
// (pairs of neighbours) or comes by shuffle (halves); other rotations load it
// once more. Beside memory it is instructions and the loads in flight: 64
// registers (50 where a warp has no more than three turns of 16-bit heads) keep
// four (five) CTAs on an SM, the warps of a CTA have equal turns, and a code is
// rounded by adding 1.5 2^23, whose low bits are then the code (a multiply-add a
// code puts them together). A group of 32 values is four neighbouring lanes: its
// extremes by two shuffles, its codes one 32-bit word of K or two 16-bit words
// of V a lane. Rotation and quantisation are in 32 bits with every step rounded
// by itself (no fused multiply-add), so the codes are those of the plain formula.
// Measured, 16384 bf16 tokens with 64 + 2 x 8 heads of 128: 158 us, 4.4 TB/s; 8192
// with 28 + 2 x 4 f16 heads 45 us (65 with eight warps of unequal turns and five
// heads a lane), rotated by halves 51; one token 2.3 us in a graph. A token's
// heads in several CTAs of three turns instead of one of five: 87 us against 80
// at 8192 tokens.
enum : int { ROPE_PAIRS, ROPE_HALVES, ROPE_ANY };

// 8 values as loaded, and as f32
template <class E> struct Raw8 { uint4 v[sizeof(E) / 2]; };
template <class E>
__device__ __forceinline__ Raw8<E> fetch8(const E* p) {
    Raw8<E> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
template <class E>
__device__ __forceinline__ void unpack8(const Raw8<E>& r, float (&x)[8]) {
    const E* e = reinterpret_cast<const E*>(r.v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<E>(e[i]);
}

// The rotation of a lane's 8 dimensions: cos and sin, of 4 pairs or of 8 values (sin with its sign)
template <int ROPE>
struct Turn {
    static constexpr int N = ROPE == ROPE_PAIRS ? 4 : 8;
    float cs[N], sn[N];
};

// FEW: a warp has at most three turns, all of them fetched at once
template <class E, class O, int D, int ROPE, bool FEW>
__global__ void __launch_bounds__(256, FEW ? 5 : 4) k_kv4_append(const __grid_constant__ fbx_kv4_cache c, const E* q, const E* k,
                                                       const E* v, int64_t ldq, int64_t ldkv, int H, int hpc,
                                                       const int32_t* __restrict__ tok_seq,
                                                       const int32_t* __restrict__ tok_pos, int rot, int neox,
                                                       const float* __restrict__ rcos, const float* __restrict__ rsin,
                                                       int n_rope, O* q_out, int64_t ldq_out, O* k_out, O* v_out,
                                                       int64_t ldkv_out) {
    using R = Kv4Rec<D>;
    constexpr int L = D / 8, HPW = 32 / L;   // lanes a head, heads a warp (D = 96: 8 lanes idle)
    constexpr int U = sizeof(E) == 4 ? 2 : FEW ? 3 : 5;
    pdl_trigger();
    const int t = blockIdx.x, HKV = c.n_head_kv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int d0 = (lane % L) * 8, half = rot / 2;
    const int h0 = hpc * blockIdx.y, h1 = min(h0 + hpc, H + 2 * HKV), step = (int)blockDim.x / 32 * HPW;
    const bool busy = lane < HPW * L, turns = d0 < rot;
    auto source = [&](int h) {
        return h < H ? q + t * ldq + h * D : h < H + HKV ? k + t * ldkv + (h - H) * D : v + t * ldkv + (h - H - HKV) * D;
    };
    pdl_wait();
    Raw8<E> raw[U];
    auto fetch = [&](int from) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = from + u * step + warp * HPW + lane / L;
            if (busy && h < h1) raw[u] = fetch8<E>(source(h) + d0);
        }
    };
    fetch(h0);
    const int pos = __ldg(tok_pos + t), seq = __ldg(tok_seq + t);
    if (pos < 0) return;   // padding
    if (seq < 0 || seq >= c.n_seqs || pos >= n_rope) {
        if (c.err && threadIdx.x == 0) atomicExch(c.err, 6);
        return;
    }
    // x0 cos - x1 sin for the first of a pair, x1 cos + x0 sin for the second
    Turn<ROPE> turn;
    const float *cr = rcos + (size_t)pos * half, *sr = rsin + (size_t)pos * half;
    if (ROPE == ROPE_ANY) {
#pragma unroll
        for (int i = 0; i < Turn<ROPE>::N; ++i) {
            const int d = d0 + i;
            const bool first = neox ? d < half : i % 2 == 0;
            const int pair = neox ? (first ? d : d - half) : d / 2;
            turn.cs[i] = d < rot ? __ldg(cr + pair) : 1.0f;
            turn.sn[i] = d < rot ? (first ? -__ldg(sr + pair) : __ldg(sr + pair)) : 0.0f;
        }
    } else if (turns) {
        const int at = ROPE == ROPE_PAIRS ? d0 / 2 : d0 < half ? d0 : d0 - half;
        const float sign = ROPE == ROPE_HALVES && d0 < half ? -1.0f : 1.0f;
#pragma unroll
        for (int i = 0; i < Turn<ROPE>::N; i += 4) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(cr + at + i)), b = __ldg(reinterpret_cast<const float4*>(sr + at + i));
            turn.cs[i] = a.x; turn.cs[i + 1] = a.y; turn.cs[i + 2] = a.z; turn.cs[i + 3] = a.w;
            turn.sn[i] = sign * b.x; turn.sn[i + 1] = sign * b.y; turn.sn[i + 2] = sign * b.z; turn.sn[i + 3] = sign * b.w;
        }
    }
    const int page = kv4_page(c, seq, pos / kKv4Page), row = pos % kKv4Page;
    if (page < 0) return;
    for (int hb = h0; hb < h1; hb += U * step) {
        if (hb > h0) fetch(hb);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (hb + u * step >= h1) break;   // the whole CTA
            const int h = hb + u * step + warp * HPW + lane / L;
            const bool live = busy && h < h1;
            const int kind = !live ? 3 : h < H ? 0 : h < H + HKV ? 1 : 2;
            float x[8];
            if (live) unpack8<E>(raw[u], x);
            else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = 0.0f;
            }
            if (ROPE == ROPE_PAIRS) {
                if (kind < 2 && turns) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const float a = x[i], b = x[i + 1], cs = turn.cs[i / 2], sn = turn.sn[i / 2];
                        x[i] = __fsub_rn(__fmul_rn(a, cs), __fmul_rn(b, sn));
                        x[i + 1] = __fadd_rn(__fmul_rn(a, sn), __fmul_rn(b, cs));
                    }
                }
            } else {
                float o[8];
                if (ROPE == ROPE_HALVES) {
                    const int from = lane + (d0 < half ? half / 8 : turns ? -(half / 8) : 0);
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, x[i], from);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int d = d0 + i, p = neox ? (d < half ? d + half : d - half) : d ^ 1;
                        o[i] = live && d < rot ? to_f32<E>(source(h)[p]) : 0.0f;
                    }
                    __syncwarp();   // every read of the head before any write: the outputs may be the inputs
                }
                if (kind < 2 && turns) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (ROPE == ROPE_HALVES || d0 + i < rot)
                            x[i] = __fadd_rn(__fmul_rn(x[i], turn.cs[i % Turn<ROPE>::N]), __fmul_rn(o[i], turn.sn[i % Turn<ROPE>::N]));
                }
            }
            if (kind == 0) store8(q_out + t * ldq_out + h * D + d0, x);
            if (!__any_sync(0xffffffffu, kind == 1 || kind == 2)) continue;
            float lo = fminf(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), fminf(fminf(x[4], x[5]), fminf(x[6], x[7])));
            float hi = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
#pragma unroll
            for (int w = 1; w <= 2; w <<= 1) {
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, w));
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, w));
            }
            if (kind != 1 && kind != 2) continue;
            if (!(lo <= hi)) lo = hi = 0.0f;   // nothing but NaN
            const __half lo16 = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
            lo = __half2float(lo16);
            const __half d16 = __float2half_rn(__fmul_rn(__fsub_rn(fminf(fmaxf(hi, -65504.0f), 65504.0f), lo), 1.0f / 15.0f));
            const float d = __half2float(d16), inv = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
            constexpr float kRound = 12582912.0f;   // 0x4B400000: 0..15 added to it stand in its low bits, rounded to even
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // clamped first (NaN to 0): the bounds are codes, so the rounding is that of the formula
                const float code = __fadd_rn(fminf(fmaxf(__fmul_rn(__fsub_rn(x[i], lo), inv), 0.0f), 15.0f), kRound);
                word += __float_as_uint(code) << (4 * i);
                x[i] = code;
            }
            constexpr uint32_t kExtra = [] {
                uint32_t e = 0;
                for (int i = 0; i < 8; ++i) e += 0x4B400000u << (4 * i);
                return e;
            }();
            word -= kExtra;
            const int hk = kind == 1 ? h - H : h - H - HKV;
            uint8_t* rec = kv4_record(c, page, hk, R::bytes);
            const int g = d0 / 32, n = (d0 / 8) % 4;
            if (kind == 1) {
                *reinterpret_cast<uint32_t*>(rec + row * R::row + 4 * R::NG * n + 4 * g) = word;
            } else {
                const int swap = ((row >> 1) & 1) * 4;
                uint8_t* at = rec + R::v + row * R::row + 2 * g;
                *reinterpret_cast<uint16_t*>(at + 2 * R::NG * ((2 * n) ^ swap)) = (uint16_t)word;
                *reinterpret_cast<uint16_t*>(at + 2 * R::NG * ((2 * n + 1) ^ swap)) = (uint16_t)(word >> 16);
            }
            if (n == 0) {
                __half* sc = reinterpret_cast<__half*>(rec + (kind == 1 ? R::kd : R::vd)) + row * R::GP + g;
                sc[0] = d16;
                sc[kKv4Page * R::GP] = lo16;
            }
            O* told = kind == 1 ? k_out : v_out;
            if (told) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __fadd_rn(lo, __fmul_rn(d, __fsub_rn(x[i], kRound)));
                store8(told + t * ldkv_out + hk * D + d0, x);
            }
        }
    }
}

// ================================================================ attention
//   s_j = scale q . k_j,  k_j = lo_jg + d_jg c_j  (g the group of a dimension)
//       = scale (sum_g d_jg (q_g . c_jg) + sum_g lo_jg sum(q_g))
//   O   = sum_j p_j v_j = sum_j (p_j d_jg) c_j + sum_j p_j lo_jg
// so the 4-bit codes themselves go through the tensor cores (mma.sync
// m16n8k16, f16 operands, exact), and scales meet sums, not values.
//
// CTA = (a run of the token's pages, kv head, up to 8 of its query heads,
// token); each of its 8 warps takes every eighth two pages of the run, one bulk
// copy a page and kv head (K and V codes and scales lie together, 2560 B at D =
// 128) into the warp's own ring of kSlots. Per page:
//   S^T[16 keys][8 heads] = K[16][D] Q^T: a k-step of 16 stays inside one
//     group, and the group's two steps' sums are scaled by d of the row;
//   O^T[16 dims][8 heads] += V^T P'^T, P' = p d per group, transposed in
//     registers (movmatrix).
// A row of an operand tile and its key differ by kv4_key (bank conflicts).
//
// What bounds it is instructions: at the full HBM rate an SM has 111 cycles for
// a page of 128 dimensions, that is 4096 values. So for 16-bit types a code is
// masked out of its word and used where it lies: bits 0..3 of a half are the f16
// subnormal c 2^-24, bits 4..7 are c 2^-20 (tensor cores take subnormals as they
// are); even dimensions' queries are 16 times as large to even that out, odd
// dimensions' outputs are 2^4 less. A product's place in the adder goes by the
// exponent field, so a subnormal keeps up to 10 bits less than a normal operand
// would: 2^-17 of the sum, against 2^-12 for f16's own rounding. f32 calls,
// which want more, take normal operands at four more instructions a word. Two
// pages a step share the waits and checks. And no maximum is formed over a
// page: the weights' reference is raised only when some lane's weight passes
// 2^kHigh, the exponent 2^E of a group's V scales only when some d passes
// 2^(E + 1); both rescale what was summed, a few times a context. With p <= 2^7
// and d 2^(7 - E) <= 2^8 the products stay in f16's range whatever the values'
// size is, and d keeps all its bits down to 2^-20 of its group's largest.
//
// Roundings: 16-bit queries go in as one f16 part, scaled by a power of two
// (exact down to 2^-23 of the head's largest), f32 ones as two (2^-22, and 2^-34
// of the head's largest), and so the sums of a group's queries. Weights p d of
// f32 calls are three bf16 parts (2^-24, in f32's range, so groups and keys of
// any size lie beside one another without an exponent), and a page's sums of
// them are added in f32. They meet codes of -8..7 with lo + 8 d in lo's place:
// sums that are all of one sign, and of which lo takes most away again, would
// leave the adder's truncation several times as large in the result. For 16 bits
// p d is rounded once, to f16. For f16 outputs it meets codes of -8..7 too (8
// sum(p d) is taken off by one more MMA a group), else that rounding would be the
// larger part of the error; for bf16, whose own step is 8 times as wide, codes
// stay 0..15 (centred ones: 53 us against 48 at 32 tokens, error against 64 bits
// 1.67e-3 against 1.74e-3, of which 1.65e-3 are the output's own rounding). In
// both a p d below 2^-14 of 2^(E - 7) is held to 2^-25 of that, where a warp's
// largest p is 2 or more.
//
// Measured at D = 128: 32 tokens of 4097-5100 bf16 keys, 64 heads in 8 groups,
// 48 us, 4.0 TB/s; 64 of 2049-2180 f16 keys, 28 heads in 4 groups, 27 us, 3.25
// TB/s (256 CTAs on 148 SMs: those with two are busy for 40000 cycles, 139 a page,
// those with one for 24000; 6000 more are the page ids, the queries and the
// merge); one of 131071 bf16 keys 41 us; one of 577 f32 keys 7.4 us, 6.6 in a
// graph; f32 at the shapes of the second and third 50 and 79 us. Tried and
// slower: equal shares of all pages for 296 CTAs (47 us at 64 x 2100), two to
// eight splits of 256 pairs (37 to 63) or of 384 (55 against 45), CTAs of four
// warps (53), scores of the next pages under this one's products.
constexpr int kAtWarps = 8, kSlots = 2;
constexpr int kMaxCluster = 8;
constexpr float kNoRef = -3.4028235e38f;   // before the first key: below every score, and finite, so that a key outside (-inf) weighs 0

// key of row r of the 16-row operand tiles
__device__ __forceinline__ int kv4_key(int r) { return (r & 8) | (r & 1 ? 4 + (((r >> 1) & 3) ^ 1) : (r >> 1) & 3); }

__device__ __forceinline__ float at_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ uint32_t b2_bits(__nv_bfloat162 b) { return *reinterpret_cast<uint32_t*>(&b); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// The 8 codes of w as f16, r[n] = (code n, code n + 4). Sub: as the subnormals
// that they are where they lie, 2^-24 for even n and 2^-20 for odd; else as
// they are (dropped into the mantissa of 1024 or of 64, which is taken off
// exactly).
template <bool Sub>
__device__ __forceinline__ void codes8(uint32_t w, uint32_t (&r)[4]) {
    if (Sub) {
        const uint32_t u = w >> 8;
        r[0] = w & 0x000F000Fu;
        r[1] = w & 0x00F000F0u;
        r[2] = u & 0x000F000Fu;
        r[3] = u & 0x00F000F0u;
    } else {
        const __half2 k1024 = bits_h2(0x64006400u), k64 = bits_h2(0x54005400u);
        const uint32_t u = w >> 8;
        r[0] = h2_bits(__hsub2(bits_h2((w & 0x000F000Fu) | 0x64006400u), k1024));
        r[1] = h2_bits(__hsub2(bits_h2((w & 0x00F000F0u) | 0x54005400u), k64));
        r[2] = h2_bits(__hsub2(bits_h2((u & 0x000F000Fu) | 0x64006400u), k1024));
        r[3] = h2_bits(__hsub2(bits_h2((u & 0x00F000F0u) | 0x54005400u), k64));
    }
}
// The same less 8, as bf16 (dropped into the mantissa of 128, which is taken off exactly together with the 8).
__device__ __forceinline__ void codes8_mid(uint32_t w, uint32_t (&r)[4]) {
    const uint32_t k136 = 0x43084308u;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const uint32_t u = (w >> 4 * n & 0x000F000Fu) | 0x43004300u;
        r[n] = b2_bits(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&k136)));
    }
}
template <int I>   // half I of a pair as f32
__device__ __forceinline__ float half_at(uint32_t u) { return I ? __high2float(bits_h2(u)) : __low2float(bits_h2(u)); }
// n words (1..4) at p, aligned to the largest power of two that divides 4 n
template <int N>
__device__ __forceinline__ void words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x; w[1] = u.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}
// the V codes of one row piece: NG 16-bit words, two a 32-bit word
template <int NG>
__device__ __forceinline__ void halves(const uint8_t* p, uint32_t (&w)[(NG + 1) / 2]) {
    if constexpr (NG == 3) {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
        w[0] = h[0] | (uint32_t)h[1] << 16;
        w[1] = h[2];
    } else {
        words<NG / 2>(p, w);
    }
}

// a / b of powers of two
__device__ __forceinline__ float over2(float a, float b) { return __int_as_float((127 << 23) + __float_as_int(a) - __float_as_int(b)); }

struct AtArgs {
    fbx_kv4_cache c;
    const void* q;
    int64_t ldq;
    int H;
    const int32_t *tok_seq, *tok_pos;
    float scale, softcap;
    int window;
    void* out;
    int64_t ldo;
    float* part;   // [token][kv head and run of 8 heads][split]: ref[8], sum[8], O[8][D], for the join; null: the splits are
                   // one cluster, which joins them through its shared memory
};

template <int D>
struct AtSmem {
    using R = Kv4Rec<D>;
    static constexpr int q = kAtWarps * kSlots * 2 * R::bytes;   // f16 queries [2 parts][8][q_row]
    static constexpr int q_row = D + 8;
    static constexpr int qs = q + 2 * 8 * q_row * 2;             // sums of a group's queries [2 parts][8][4] f16
    static constexpr int ex = qs + 2 * 8 * 4 * 2;              // the heads' exponents as factors [8]
    static constexpr int bar = ex + 32;
    static constexpr int bytes = bar + 8 * kAtWarps * kSlots;
    // at the end, over the rings: [warps][8] ref, [warps][8] sum, [warps][8][D + 4] O
    static constexpr int ml = 0, o = kAtWarps * 8 * 8;
    static constexpr int part = o + kAtWarps * 8 * (D + 4) * 4;   // and of the CTA, as AtArgs::part
    static_assert(part + (16 + 8 * D) * 4 <= q, "merge area");
};

// how the weights of an element type go into the products with V (see above)
enum : int { W_PARTS, W_MID, W_CODE };
template <class E> struct AtWeights { static constexpr int mode = W_PARTS; };
template <> struct AtWeights<__half> { static constexpr int mode = W_MID; };
template <> struct AtWeights<__nv_bfloat16> { static constexpr int mode = W_CODE; };

template <class E, int D>
__global__ void __launch_bounds__(32 * kAtWarps, 2) k_kv4_attention(const __grid_constant__ AtArgs A) {
    using R = Kv4Rec<D>;
    using M = AtSmem<D>;
    constexpr int NG = R::NG, GP = R::GP, PL = sizeof(E) == 4 ? 2 : 1, W = AtWeights<E>::mode;
    constexpr bool SUB = W != W_PARTS;
    // a weight passes 2^kHigh: the reference becomes the largest score less kTo
    constexpr float kHigh = SUB ? 7.0f : 14.0f, kTo = SUB ? 1.0f : 8.0f;
    constexpr float kCode = SUB ? 1048576.0f : 1.0f;   // a code over its operand
    extern __shared__ __align__(128) uint8_t sm[];
    const fbx_kv4_cache& c = A.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int tok = blockIdx.z, G = A.H / c.n_head_kv, runs = (G + 7) / 8;
    const int hk = blockIdx.y / runs, g0 = blockIdx.y % runs * 8, gn = min(8, G - g0), S = gridDim.x;
    uint64_t* bar = reinterpret_cast<uint64_t*>(sm + M::bar) + warp * kSlots;
    uint8_t* ring = sm + warp * kSlots * 2 * R::bytes;
    pdl_trigger();
    if (lane < kSlots) mbar_init(&bar[lane], 2);
    mbar_fence_init();
    pdl_wait();
    // everything that depends on nothing else at once: the token's place and this warp's query head
    const int pos = __ldg(A.tok_pos + tok), seq = __ldg(A.tok_seq + tok);
    static_assert(kAtWarps == 8, "a warp a query head");
    float x[NG];
#pragma unroll
    for (int e = 0; e < NG; ++e)
        x[e] = warp < gn ? to_f32<E>(static_cast<const E*>(A.q)[tok * A.ldq + (int64_t)(hk * G + g0 + warp) * D + 32 * e + lane]) : 0.0f;
    if (pos < 0) return;   // padding
    const bool known = seq >= 0 && seq < c.n_seqs;
    if (!known && c.err && threadIdx.x == 0) atomicExch(c.err, 6);

    // this warp's steps of two neighbouring pages: step j has the pages first + 16 j and the next, below last;
    // lane l holds the page l & 1 of its (l / 2)-th step (of 16)
    const int key0 = A.window > 0 ? max(0, pos - A.window + 1) : 0;
    const int p0 = key0 / kKv4Page, p1 = min(pos / kKv4Page + 1, c.table_stride);
    if (pos / kKv4Page >= c.table_stride && c.err && threadIdx.x == 0) atomicExch(c.err, 6);
    const int per = (max(p1 - p0, 0) + S - 1) / S;
    const int first = p0 + blockIdx.x * per + 2 * warp, last = min(p0 + ((int)blockIdx.x + 1) * per, p1);
    const int n = known && first < last ? (last - first + 2 * kAtWarps - 1) / (2 * kAtWarps) : 0;
    auto look_up = [&](int j0) {
        const int i = first + (j0 + lane / 2) * 2 * kAtWarps + (lane & 1);
        return j0 + lane / 2 < n && i < last ? kv4_page(c, seq, i) : -1;
    };
    int ids = look_up(0), ids_next = -1;
    __syncwarp();
    auto issue = [&](int j, int id) {   // lanes 0 and 1 bring a page each; without one the barrier's phase passes without it
        const int page = __shfl_sync(0xffffffffu, id, 2 * (j & 15) + (lane & 1));
        if (lane < 2) {
            uint64_t* b = &bar[j % kSlots];
            if (page >= 0) {
                mbar_expect_tx(b, R::bytes);
                bulk_g2s(ring + ((j % kSlots) * 2 + lane) * R::bytes, kv4_record(c, page, hk, R::bytes), R::bytes, b);
            } else {
                mbar_arrive(b);
            }
        }
    };
    for (int j = 0; j < kSlots && j < n; ++j) issue(j, ids);

    // the queries: warp w brings head g0 + w to 2^9 .. 2^10 in size (16 times that, and sums of 32, are still f16), as f16 parts,
    // dimensions 32 e + 8 t + n in the order (0, 4), (1, 5), (2, 6), (3, 7) of n that a lane's operands have
    constexpr int QS = AtSmem<D>::q_row;
    {
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < NG; ++e) top = fmaxf(top, fabsf(x[e]));
        top = warp_max(top);
        int ex = (int)(__float_as_uint(top) >> 23) - 127;
        if (ex == 128 || top == 0.0f) ex = 0;
        ex = max(ex, -110) - 9;
        const float down = __int_as_float((127 - ex) << 23);
        __half* sq = reinterpret_cast<__half*>(sm + M::q) + warp * QS + (lane & 24) + 2 * (lane & 3) + (lane >> 2 & 1);
        __half* ss = reinterpret_cast<__half*>(sm + M::qs) + warp * 4;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < NG; ++e) {
            sum[e] = x[e] * down;
            const float z = SUB && lane % 2 == 0 ? 16.0f * sum[e] : sum[e];   // a code of an even dimension is 2^-4 less
            const __half hi = __float2half_rn(z);
            sq[32 * e] = hi;
            if (PL == 2) sq[8 * QS + 32 * e] = __float2half_rn(z - __half2float(hi));
        }
#pragma unroll
        for (int w = 16; w > 0; w >>= 1)
#pragma unroll
            for (int e = 0; e < NG; ++e) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], w);
        if (lane == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const __half h = __float2half_rn(sum[e]);
                ss[e] = h;
                ss[32 + e] = __float2half_rn(sum[e] - __half2float(h));
            }
            reinterpret_cast<float*>(sm + M::ex)[warp] = __int_as_float((127 + ex) << 23);
        }
    }
    __syncthreads();
    // B operands of the scores
    uint32_t qb[NG][4];
#pragma unroll
    for (int e = 0; e < NG; ++e) words<4>(sm + M::q + (g * QS + 32 * e + 8 * t) * 2, qb[e]);
    // and of sum_g lo sum(q_g): the sums' high parts against k = 0..3, their low parts against k = 4..7
    const uint32_t qsb = *reinterpret_cast<const uint32_t*>(sm + M::qs + (t >> 1) * 64 + g * 8 + (t & 1) * 4);
    constexpr float kLog2e = 1.4426950408889634f;
    float cs[2];   // log2 units of the heads 2 t, 2 t + 1
    const bool cap = A.softcap > 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        cs[i] = A.scale * reinterpret_cast<const float*>(sm + M::ex)[2 * t + i] * (cap ? 1.0f / A.softcap : kLog2e);
    float ref[2] = {kNoRef, kNoRef}, sum[2] = {0.0f, 0.0f};
    __half2 down_e[GP / 2];   // 2^(7 - E) of the groups 2 e, 2 e + 1, E from -8 on
#pragma unroll
    for (int e = 0; e < GP / 2; ++e) down_e[e] = bits_h2(0x78007800u);   // 2^15
    // O^T 2^(7 - E) / kCode (O^T for f32 calls): dims 32 e + 4 g + 2 u (accumulators 0, 1) and the next (2, 3), heads 2 t + (0, 1)
    // mid: -8 sum(p d) 2^(7 - E) / (16 kCode) of the groups 2 e (accumulators 0, 1) and 2 e + 1 (2, 3)
    float o[NG][2][4], olo[NG][2], mid[GP / 2][4];
#pragma unroll
    for (int e = 0; e < NG; ++e) {
        olo[e][0] = olo[e][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[e][0][i] = o[e][1][i] = 0.0f;
            if (W == W_MID) mid[e / 2][i] = 0.0f;
        }
    }
    const int row = kv4_key(g);   // and row + 8
    const int vrow = kv4_key(2 * t), vrow2 = kv4_key(2 * t + 1), piece = 2 * NG * (g ^ ((vrow & 2) << 1));
    bool ok = true;
    const int lrow = 4 * (t & 1);
    const bool lhas = 2 * (t & 1) < GP;
    const uint32_t lkeep = NG == 3 && (t & 1) ? 0xFFFFu : 0xFFFFFFFFu;   // not the padding
    int j = 0;
    for (; j < n; ++j) {
        if ((j & 15) == 16 - kSlots) ids_next = look_up((j & ~15) + 16);
        const uint32_t parity = (uint32_t)(j / kSlots) & 1u;
        ok = __all_sync(0xffffffffu, mbar_wait_soon(&bar[j % kSlots], parity));
        if (!ok) break;
        const uint8_t* rec0 = ring + (j % kSlots) * 2 * R::bytes;
        // ---- scores of keys row and row + 8 (0, 1 and 2, 3) of both pages, heads 2 t, 2 t + 1, in log2 units
        float s[2][4];
        uint32_t v0[2][GP / 2], v1[2][GP / 2], u0[2][GP / 2], u1[2][GP / 2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint8_t* rec = rec0 + h * R::bytes;
            const uint32_t l0 = lhas ? *reinterpret_cast<const uint32_t*>(rec + R::klo + row * GP * 2 + lrow) & lkeep : 0u;
            const uint32_t l1 = lhas ? *reinterpret_cast<const uint32_t*>(rec + R::klo + (row + 8) * GP * 2 + lrow) & lkeep : 0u;
            uint32_t w0[NG], w1[NG], d0[GP / 2], d1[GP / 2];
            words<NG>(rec + row * R::row + 4 * NG * t, w0);
            words<NG>(rec + (row + 8) * R::row + 4 * NG * t, w1);
            words<GP / 2>(rec + R::kd + row * GP * 2, d0);
            words<GP / 2>(rec + R::kd + (row + 8) * GP * 2, d1);
            float sl[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma8(sl, l0, l1, qsb);
#pragma unroll
            for (int e = 0; e < NG; ++e) {
                uint32_t a[4], b[4];
                codes8<SUB>(w0[e], a);
                codes8<SUB>(w1[e], b);
                float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma16(x, a[0], b[0], a[1], b[1], qb[e][0], qb[e][1]);
                mma16(x, a[2], b[2], a[3], b[3], qb[e][2], qb[e][3]);
                if (PL == 2) {   // the low parts stay in shared memory: registers are full
                    uint32_t ql[4];
                    words<4>(sm + M::q + ((8 + g) * QS + 32 * e + 8 * t) * 2, ql);
                    mma16(x, a[0], b[0], a[1], b[1], ql[0], ql[1]);
                    mma16(x, a[2], b[2], a[3], b[3], ql[2], ql[3]);
                }
                const float da = e & 1 ? half_at<1>(d0[e / 2]) : half_at<0>(d0[e / 2]);
                const float db = e & 1 ? half_at<1>(d1[e / 2]) : half_at<0>(d1[e / 2]);
                s[h][0] = e ? fmaf(da, x[0], s[h][0]) : da * x[0];
                s[h][1] = e ? fmaf(da, x[1], s[h][1]) : da * x[1];
                s[h][2] = e ? fmaf(db, x[2], s[h][2]) : db * x[2];
                s[h][3] = e ? fmaf(db, x[3], s[h][3]) : db * x[3];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[h][i] = fmaf(s[h][i], kCode, sl[i]) * cs[i & 1];
            words<GP / 2>(rec + R::vd + row * GP * 2, v0[h]);
            words<GP / 2>(rec + R::vd + (row + 8) * GP * 2, v1[h]);
            words<GP / 2>(rec + R::vlo + row * GP * 2, u0[h]);
            words<GP / 2>(rec + R::vlo + (row + 8) * GP * 2, u1[h]);
            if (NG == 3) v0[h][1] &= 0xFFFFu, v1[h][1] &= 0xFFFFu;
        }
        if (cap) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i / 4][i % 4] = A.softcap * kLog2e * tanhf(s[i / 4][i % 4]);
        }
        // ---- at the edges of what the token sees, and where there is no page: keys outside have no weight and no scale
        const int i0 = first + j * 2 * kAtWarps, kb = i0 * kKv4Page;
        const unsigned here = __ballot_sync(0xffffffffu, ids >= 0) >> (2 * (j & 15));
        if (kb + 2 * kKv4Page - 1 > pos || kb < key0 || (here & 3) != 3) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = kb + h * kKv4Page + row;
                const bool page = here >> h & 1, in0 = page && key <= pos && key >= key0, in1 = page && key + 8 <= pos && key + 8 >= key0;
                if (!in0) s[h][0] = s[h][1] = -INFINITY;
                if (!in1) s[h][2] = s[h][3] = -INFINITY;
#pragma unroll
                for (int e = 0; e < GP / 2; ++e) {
                    v0[h][e] = in0 ? v0[h][e] : 0u;
                    u0[h][e] = in0 ? u0[h][e] : 0u;
                    v1[h][e] = in1 ? v1[h][e] : 0u;
                    u1[h][e] = in1 ? u1[h][e] : 0u;
                }
            }
        }
        // ---- the references, raised when a weight passes 2^kHigh or a d passes 2^(E + 1)
        __half2 dm[GP / 2];
        bool wide = false;
        if (SUB) {
#pragma unroll
            for (int e = 0; e < GP / 2; ++e) {
                dm[e] = __hmax2(__hmax2(bits_h2(v0[0][e]), bits_h2(v1[0][e])), __hmax2(bits_h2(v0[1][e]), bits_h2(v1[1][e])));
                wide |= !__hble2(__hmul2(dm[e], down_e[e]), bits_h2(0x5C005C00u));   // 2^8
            }
        }
        const float mx0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2]));
        const float mx1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
        const bool high = fmaxf(mx0 - ref[0], mx1 - ref[1]) > kHigh;
        if (__any_sync(0xffffffffu, wide || high)) {
            if (SUB && __any_sync(0xffffffffu, wide)) {
#pragma unroll
                for (int e2 = 0; e2 < GP / 2; ++e2) {
#pragma unroll
                    for (int w = 4; w <= 16; w <<= 1) dm[e2] = __hmax2(dm[e2], bits_h2(__shfl_xor_sync(0xffffffffu, h2_bits(dm[e2]), w)));
                    float down[2] = {__low2float(down_e[e2]), __high2float(down_e[e2])};
                    const float d[2] = {__low2float(dm[e2]), __high2float(dm[e2])};
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int e = 2 * e2 + i;
                        if (e >= NG || !(d[i] * down[i] > 256.0f)) continue;
                        // d < 2^E, so that the ones to come seldom raise E again
                        const int E = (int)(__float_as_uint(d[i]) >> 23) - 127 + 1;
                        const float to = __int_as_float((127 + 7 - E) << 23), f = over2(to, down[i]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            o[e][0][k] *= f;
                            o[e][1][k] *= f;
                        }
                        if (W == W_MID) mid[e2][2 * i] *= f, mid[e2][2 * i + 1] *= f;
                        down[i] = to;
                    }
                    down_e[e2] = __floats2half2_rn(down[0], down[1]);
                }
            }
            if (__any_sync(0xffffffffu, high)) {
                float mx[2] = {mx0, mx1}, f[2];
#pragma unroll
                for (int w = 4; w <= 16; w <<= 1) {
                    mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], w));
                    mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], w));
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float to = mx[i] - ref[i] > kHigh ? mx[i] - kTo : ref[i];
                    f[i] = to == ref[i] ? 1.0f : at_ex2(ref[i] - to);
                    ref[i] = to;
                    sum[i] *= f[i];
                }
#pragma unroll
                for (int e = 0; e < NG; ++e) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[e][0][i] *= f[i & 1];
                        o[e][1][i] *= f[i & 1];
                    }
                    if (W == W_MID) mid[e / 2][2 * (e & 1)] *= f[0], mid[e / 2][2 * (e & 1) + 1] *= f[1];
                    olo[e][0] *= f[0];
                    olo[e][1] *= f[1];
                }
            }
        }
        // ---- d 2^(7 - E), or d, in d's place; one below 0 has codes of 0 only (f16 rounded the group's minimum up past its
        // maximum) and counts as 0
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < GP / 2; ++e) {
                const __half2 a = bits_h2(v0[h][e]), b = bits_h2(v1[h][e]), zero = bits_h2(0u);
                v0[h][e] = h2_bits(SUB ? __hfma2_relu(a, down_e[e], zero) : __hmax2_nan(a, zero));
                v1[h][e] = h2_bits(SUB ? __hfma2_relu(b, down_e[e], zero) : __hmax2_nan(b, zero));
            }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = at_ex2(s[h][i] - ref[i & 1]);
            sum[0] += p[0] + p[2];
            sum[1] += p[1] + p[3];
            // ---- V: pairs of keys (2 t, 2 t + 1) and (2 t + 8, 2 t + 9) of the tile, 4 dims a group
            uint32_t va[(NG + 1) / 2], vb[(NG + 1) / 2], vc[(NG + 1) / 2], vd[(NG + 1) / 2];
            const uint8_t* vr = rec0 + h * R::bytes + R::v + piece;
            halves<NG>(vr + vrow * R::row, va);
            halves<NG>(vr + vrow2 * R::row, vb);
            halves<NG>(vr + (vrow + 8) * R::row, vc);
            halves<NG>(vr + (vrow2 + 8) * R::row, vd);
#pragma unroll
            for (int e = 0; e < NG; ++e) {
                const float da = e & 1 ? half_at<1>(v0[h][e / 2]) : half_at<0>(v0[h][e / 2]);
                const float db = e & 1 ? half_at<1>(v1[h][e / 2]) : half_at<0>(v1[h][e / 2]);
                float la = e & 1 ? half_at<1>(u0[h][e / 2]) : half_at<0>(u0[h][e / 2]);
                float lb = e & 1 ? half_at<1>(u1[h][e / 2]) : half_at<0>(u1[h][e / 2]);
                if (W != W_CODE) {
                    // 8, or 8 2^(E - 7): the exponents of that and of 2^(7 - E) add up to 3
                    const float k = W == W_MID ? (e & 1 ? half_at<1>(0x84008400u - h2_bits(down_e[e / 2])) : half_at<0>(0x84008400u - h2_bits(down_e[e / 2]))) : 8.0f;
                    la = fmaf(k, da, la);
                    lb = fmaf(k, db, lb);
                }
                olo[e][0] = fmaf(p[0], la, fmaf(p[2], lb, olo[e][0]));
                olo[e][1] = fmaf(p[1], la, fmaf(p[3], lb, olo[e][1]));
                uint32_t ra[4], rc[4];
                const uint32_t wa = __byte_perm(va[e / 2], vb[e / 2], e & 1 ? 0x7632 : 0x5410);
                const uint32_t wc = __byte_perm(vc[e / 2], vd[e / 2], e & 1 ? 0x7632 : 0x5410);
                if constexpr (W == W_PARTS) {
                    codes8_mid(wa, ra);
                    codes8_mid(wc, rc);
                    // a page's sums start at 0 and are added in f32: sums over a long context in the tensor core, whose additions cut
                    // off, would all come out a little small (4e-5 after 16000 keys of a warp)
                    float x[4] = {p[0] * da, p[1] * da, p[2] * db, p[3] * db}, y[2][4] = {};
#pragma unroll
                    for (int part = 0; part < 3; ++part) {
                        const __nv_bfloat162 z0 = __floats2bfloat162_rn(x[0], x[1]), z1 = __floats2bfloat162_rn(x[2], x[3]);
                        const uint32_t b0 = transpose8(b2_bits(z0)), b1 = transpose8(b2_bits(z1));
#pragma unroll
                        for (int u = 0; u < 2; ++u) mma16_bf16(y[u], ra[2 * u], ra[2 * u + 1], rc[2 * u], rc[2 * u + 1], b0, b1);
                        x[0] -= __low2float(z0);
                        x[1] -= __high2float(z0);
                        x[2] -= __low2float(z1);
                        x[3] -= __high2float(z1);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[e][0][i] += y[0][i];
                        o[e][1][i] += y[1][i];
                    }
                    continue;
                }
                codes8<SUB>(wa, ra);
                codes8<SUB>(wc, rc);
                const __half2 hi0 = __floats2half2_rn(p[0] * da, p[1] * da), hi1 = __floats2half2_rn(p[2] * db, p[3] * db);
                const uint32_t b0 = transpose8(h2_bits(hi0)), b1 = transpose8(h2_bits(hi1));
#pragma unroll
                for (int u = 0; u < 2; ++u) mma16(o[e][u], ra[2 * u], ra[2 * u + 1], rc[2 * u], rc[2 * u + 1], b0, b1);
                if (W == W_MID) {   // -8 in the upper or lower 8 rows
                    const uint32_t a = e & 1 ? 0u : 0x80088008u, b = e & 1 ? 0x80088008u : 0u;
                    mma16(mid[e / 2], a, b, a, b, b0, b1);
                }
            }
        }
        __syncwarp();   // the slot is read
        if (j + kSlots < n) issue(j + kSlots, ((j + kSlots) & ~15) == (j & ~15) ? ids : ids_next);
        if ((j & 15) == 15) ids = ids_next;
    }
    if (!ok) {   // a copy did not arrive in time: it and the one behind it may still be under way, and nobody gets an answer
        for (int k = j; k < j + kSlots && k < n; ++k) mbar_wait_bounded(&bar[k % kSlots], (uint32_t)(k / kSlots) & 1u);
        sum[0] = sum[1] = NAN;
        if (c.err && lane == 0) atomicExch(c.err, 7);
    }
    // ---- the lanes' sums over keys (those of other g), then the warps
#pragma unroll
    for (int w = 4; w <= 16; w <<= 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], w);
#pragma unroll
            for (int e = 0; e < NG; ++e) olo[e][i] += __shfl_xor_sync(0xffffffffu, olo[e][i], w);
        }
    }
    __syncthreads();   // every ring is done with
    float* ml = reinterpret_cast<float*>(sm + M::ml);
    float* so = reinterpret_cast<float*>(sm + M::o);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int h = 2 * t + i;
        if (g == 0) {
            ml[warp * 8 + h] = ref[i];
            ml[8 * kAtWarps + warp * 8 + h] = sum[i];
        }
#pragma unroll
        for (int e = 0; e < NG; ++e) {
            // odd and even dimensions
            const float up = SUB ? over2(kCode, half_at<0>(h2_bits(down_e[e / 2]) >> (e & 1 ? 16 : 0))) : 1.0f, ev = SUB ? 16.0f * up : up;
            const float lo = olo[e][i] + (W == W_MID ? ev * mid[e / 2][2 * (e & 1) + i] : 0.0f);
            *reinterpret_cast<float4*>(so + (warp * 8 + h) * (D + 4) + 32 * e + 4 * g) =
                make_float4(fmaf(ev, o[e][0][i], lo), fmaf(up, o[e][0][2 + i], lo), fmaf(ev, o[e][1][i], lo), fmaf(up, o[e][1][2 + i], lo));
        }
    }
    __syncthreads();
    float* part = reinterpret_cast<float*>(sm + M::part);
    if (A.part) part = A.part + ((size_t)(tok * gridDim.y + blockIdx.y) * S + blockIdx.x) * (16 + 8 * D);
    for (int i = threadIdx.x; i < gn * (D / 4); i += 32 * kAtWarps) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float top = -INFINITY, l = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kAtWarps; ++w) top = fmaxf(top, ml[w * 8 + h]);
#pragma unroll
        for (int w = 0; w < kAtWarps; ++w) {
            const float f = at_ex2(ml[w * 8 + h] - top);
            const float4 y = *reinterpret_cast<const float4*>(so + (w * 8 + h) * (D + 4) + d);
            l = fmaf(f, ml[8 * kAtWarps + w * 8 + h], l);
            x.x = fmaf(f, y.x, x.x);
            x.y = fmaf(f, y.y, x.y);
            x.z = fmaf(f, y.z, x.z);
            x.w = fmaf(f, y.w, x.w);
        }
        if (A.part || S > 1) {
            if (d == 0) {
                part[h] = top;
                part[8 + h] = l;
            }
            *reinterpret_cast<float4*>(part + 16 + h * D + d) = x;
        } else {
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;   // NaN stays NaN
            store4(static_cast<E*>(A.out) + tok * A.ldo + (int64_t)(hk * G + g0 + h) * D + d, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        }
    }
    if (A.part || S == 1) return;
    // ---- one cluster: every CTA joins its part of the outputs
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int i = threadIdx.x + 32 * kAtWarps * blockIdx.x; i < gn * (D / 4); i += 32 * kAtWarps * S) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float tops[kMaxCluster], top = -INFINITY, l = 0.0f;
        float4 y[kMaxCluster], x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int s = 0; s < kMaxCluster; ++s) {
            const float* p = cluster.map_shared_rank(part, s < S ? s : 0);
            tops[s] = s < S ? p[h] : -INFINITY;
            y[s] = *reinterpret_cast<const float4*>(p + 16 + h * D + d);
            top = fmaxf(top, tops[s]);
        }
#pragma unroll
        for (int s = 0; s < kMaxCluster; ++s) {
            if (s >= S) break;
            const float f = at_ex2(tops[s] - top);
            l = fmaf(f, cluster.map_shared_rank(part, s)[8 + h], l);
            x.x = fmaf(f, y[s].x, x.x);
            x.y = fmaf(f, y[s].y, x.y);
            x.z = fmaf(f, y[s].z, x.z);
            x.w = fmaf(f, y[s].w, x.w);
        }
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;   // NaN stays NaN
        store4(static_cast<E*>(A.out) + tok * A.ldo + (int64_t)(hk * G + g0 + h) * D + d, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    }
    cluster.sync();   // nobody's shared memory goes while it is read
}

// The splits of one (token, query head) joined: out = sum_s 2^(ref_s - top) O_s / sum_s 2^(ref_s - top) sum_s.
// Warp w takes the splits w, w + 8, .., a lane D / 32 dimensions; the loads do not wait for the reference. Latency: 3 us of the
// 39 at 131071 keys, 37 splits.
constexpr int kJoinWarps = 8;
template <class E, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) k_kv4_join(const float* __restrict__ part, int S, int H, int HKV,
                                                              const int32_t* __restrict__ tok_pos, E* out, int64_t ldo) {
    constexpr int N = D / 32, U = 5;   // U splits of a warp in flight
    pdl_trigger();
    pdl_wait();
    const int tok = blockIdx.y, h = blockIdx.x, G = H / HKV, runs = (G + 7) / 8, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (tok_pos[tok] < 0) return;
    const int hg = h % G, r = hg % 8;
    const float* p = part + (size_t)(tok * HKV * runs + h / G * runs + hg / 8) * S * (16 + 8 * D);
    __shared__ float st[kJoinWarps], sl[kJoinWarps], so[kJoinWarps][D];
    float top = -INFINITY, l = 0.0f, o[N];
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = 0.0f;
    for (int s0 = warp; s0 < S; s0 += kJoinWarps * U) {
        float ref[U], sum[U], x[U][N], up = top;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * kJoinWarps;
            const float* ps = p + (size_t)s * (16 + 8 * D);
            ref[u] = s < S ? ps[r] : -INFINITY;
            sum[u] = s < S ? ps[8 + r] : 0.0f;
#pragma unroll
            for (int e = 0; e < N; ++e) x[u][e] = s < S ? ps[16 + r * D + 32 * e + lane] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) up = fmaxf(up, ref[u]);
        const float f0 = at_ex2(top - up);
        l *= f0;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] *= f0;
        top = up;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float f = at_ex2(ref[u] - top);
            l = fmaf(f, sum[u], l);
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] = fmaf(f, x[u][e], o[e]);
        }
    }
    if (lane == 0) {
        st[warp] = top;
        sl[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) so[warp][32 * e + lane] = o[e];
    __syncthreads();
    if (threadIdx.x < D) {
        top = -INFINITY;
        l = 0.0f;
        float y = 0.0f;
        for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, st[w]);
        for (int w = 0; w < kJoinWarps; ++w) {
            const float f = at_ex2(st[w] - top);
            l = fmaf(f, sl[w], l);
            y = fmaf(f, so[w][threadIdx.x], y);
        }
        out[tok * ldo + (int64_t)h * D + threadIdx.x] = from_f32<E>(l != 0.0f ? y / l : 0.0f);
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

template <class E, class O, int D, int ROPE>
static cudaError_t launch_append_as(const AppendArgs& a, cudaStream_t st) {
    constexpr int HPW = 32 / (D / 8);
    const int H = a.q ? a.H : 0, heads = H + 2 * a.c.n_head_kv;
    // few tokens: CTAs of 8 warps with a turn each; many: a token's heads in one CTA, of as many warps as have equal turns
    const int groups = (heads + HPW - 1) / HPW, turns = (groups + 7) / 8;
    const bool many = a.T >= 148;
    const int warps = many ? (groups + turns - 1) / turns : std::min(8, groups), hpc = many ? heads : warps * HPW;
    const bool few = sizeof(E) == 2 && turns <= 3;
    auto kern = few ? k_kv4_append<E, O, D, ROPE, sizeof(E) == 2> : k_kv4_append<E, O, D, ROPE, false>;
    return fbk_launch_early(kern, dim3(a.T, (heads + hpc - 1) / hpc), dim3(32 * warps), 0, st, 1, a.c,
                            (const E*)a.q, (const E*)a.k, (const E*)a.v, a.ldq, a.ldkv, H, hpc, a.tok_seq, a.tok_pos, a.rot,
                            a.neox, a.rcos, a.rsin, a.n_rope, (O*)a.q_out, a.ldq_out, (O*)a.k_out, (O*)a.v_out, a.ldkv_out);
}
template <class E, class O, int D>
static cudaError_t launch_append(const AppendArgs& a, cudaStream_t st) {
    // whole lanes of 8 dimensions, and tables that can be read 16 bytes at a time
    const bool wide = ((reinterpret_cast<uintptr_t>(a.rcos) | reinterpret_cast<uintptr_t>(a.rsin)) & 15) == 0;
    return wide && !a.neox && a.rot % 8 == 0 ? launch_append_as<E, O, D, ROPE_PAIRS>(a, st)
         : wide && a.neox && a.rot % 16 == 0 ? launch_append_as<E, O, D, ROPE_HALVES>(a, st)
                                             : launch_append_as<E, O, D, ROPE_ANY>(a, st);
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

// CTAs a token and kv head: as many as two an SM give, each warp of them with a step or more. Up to eight are one cluster (2,
// 4 or 8 of them) and one launch; more leave partial results for a second one.
static int at_splits(int T, int H, int HKV, int max_keys) {
    constexpr int64_t kRoom = 2 * 148;
    const int64_t pairs = (int64_t)T * HKV * ((H / HKV + 7) / 8);
    const int pages = (max_keys - 1) / kKv4Page + 1;
    const int S = (int)std::max<int64_t>(1, std::min<int64_t>(kRoom / pairs, (pages + 2 * kAtWarps - 1) / (2 * kAtWarps)));
    if (S > kMaxCluster) return S;
    int c = 1;
    while (c < S) c *= 2;
    return c > S && pairs * c > kRoom ? c / 2 : c;
}

template <class E, int D>
static cudaError_t launch_kv4_attention(const AtArgs& a, int T, int S, cudaStream_t st) {
    using M = AtSmem<D>;
    static uint64_t set = 0;   // one bit a device; setting it twice does no harm
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (!(__atomic_load_n(&set, __ATOMIC_RELAXED) >> (dev & 63) & 1)) {
        e = cudaFuncSetAttribute(k_kv4_attention<E, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, M::bytes);
        if (e != cudaSuccess) return e;
        __atomic_fetch_or(&set, (uint64_t)1 << (dev & 63), __ATOMIC_RELAXED);
    }
    const int HKV = a.c.n_head_kv;
    const dim3 grid(S, HKV * ((a.H / HKV + 7) / 8), T);
    e = fbk_launch_early(k_kv4_attention<E, D>, grid, dim3(32 * kAtWarps), (size_t)M::bytes, st, a.part ? 1 : S, a);
    if (e != cudaSuccess || !a.part) return e;
    return fbk_launch_early(k_kv4_join<E, D>, dim3(a.H, T), dim3(32 * kJoinWarps), 0, st, 1, (const float*)a.part, S, a.H, HKV, a.tok_pos, (E*)a.out, a.ldo);
}
template <class E>
static cudaError_t kv4_attention_d(const AtArgs& a, int T, int S, cudaStream_t st) {
    return a.c.head_dim == 128 ? launch_kv4_attention<E, 128>(a, T, S, st)
         : a.c.head_dim == 96 ? launch_kv4_attention<E, 96>(a, T, S, st) : launch_kv4_attention<E, 64>(a, T, S, st);
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

extern "C" size_t fbk_kv4_attention_workspace(int T, int H, int HKV, int D, int max_keys) {
    const int S = at_splits(T, H, HKV, max_keys);
    return S > kMaxCluster ? (size_t)T * HKV * ((H / HKV + 7) / 8) * S * (16 + 8 * D) * sizeof(float) : 0;
}

extern "C" int fbk_kv4_attention(const fbx_kv4_cache& c, int type, const void* q, int64_t ldq, int T, int H,
                                 const int32_t* tok_seq, const int32_t* tok_pos, int max_keys, float scale, float softcap,
                                 int window, void* out, int64_t ldo, void* ws, cudaStream_t st) {
    // a window bounds the keys too (it may begin inside a page); never more splits than the workspace was sized for
    const int keys = window > 0 ? (int)std::min<int64_t>(max_keys, (int64_t)window + kKv4Page) : max_keys;
    const int S = at_splits(T, H, c.n_head_kv, keys);
    const AtArgs a{c, q, ldq, H, tok_seq, tok_pos, scale, softcap, window, out, ldo, S > kMaxCluster ? (float*)ws : nullptr};
    return (int)(type == T_F32 ? kv4_attention_d<float>(a, T, S, st)
               : type == T_F16 ? kv4_attention_d<__half>(a, T, S, st) : kv4_attention_d<__nv_bfloat16>(a, T, S, st));
}
