// kv4.cuh — the paged cache held in 4 bits: record layout and element types.
//
// The layout (fish_kernels.h states it byte by byte) is the one in which a
// warp's lanes read their MMA operands as wide words: of a K row, lane 4 g + t
// takes the dimensions 32 g' + 8 t + (0..7) of every group g', one 32-bit word
// a group, adjacent in memory; of a V row, lane 4 h + t takes the dimensions
// 32 g' + 4 h + (0..3), one 16-bit word a group. The V pieces of rows with bit
// 1 set are swapped by halves, so that the four rows read together fall on
// different shared-memory banks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"
#include "fish/fish_kernels.h"

namespace fb {

constexpr int kKv4Page = 16;

template <int D>
struct Kv4Rec {
    static constexpr int NG = D / 32;            // groups of 32 values
    static constexpr int GP = (NG + 1) / 2 * 2;  // scales a row, padded
    static constexpr int row = D / 2;            // bytes of codes a row
    static constexpr int codes = kKv4Page * row;
    static constexpr int scales = kKv4Page * GP * 2;
    static constexpr int kd = codes, klo = codes + scales;
    static constexpr int v = codes + 2 * scales, vd = v + codes, vlo = vd + scales;
    static constexpr int bytes = 2 * v;
};

// page of position 16 i of sequence s, or -1 (flagged) when the tables do not hold it
__device__ __forceinline__ int kv4_page(const fbx_kv4_cache& c, int s, int i) {
    if (i >= c.table_stride) {
        if (c.err) atomicExch(c.err, 6);
        return -1;
    }
    const int p = __ldg(c.page_table + (size_t)s * c.table_stride + i);
    if (p < 0 || p >= c.n_pages) {
        if (c.err) atomicExch(c.err, 5);
        return -1;
    }
    return p;
}
__device__ __forceinline__ uint8_t* kv4_record(const fbx_kv4_cache& c, int page, int head, int rec_bytes) {
    return static_cast<uint8_t*>(c.pool) + (size_t)page * c.page_stride + c.layer_offset + (size_t)head * rec_bytes;
}

// element types of device buffers
template <class E> __device__ __forceinline__ float to_f32(E x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class E> __device__ __forceinline__ E from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 8 consecutive values at a 16-byte boundary
template <class E>
__device__ __forceinline__ void store8(E* p, const float (&x)[8]) {
    if constexpr (sizeof(E) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint4 raw;
        E* e = reinterpret_cast<E*>(&raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f32<E>(x[i]);
        *reinterpret_cast<uint4*>(p) = raw;
    }
}

// 4 consecutive values at a boundary of 4
template <class E>
__device__ __forceinline__ void store4(E* p, float a, float b, float c, float d) {
    if constexpr (sizeof(E) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
    } else {
        uint2 raw;
        E* e = reinterpret_cast<E*>(&raw);
        e[0] = from_f32<E>(a);
        e[1] = from_f32<E>(b);
        e[2] = from_f32<E>(c);
        e[3] = from_f32<E>(d);
        *reinterpret_cast<uint2*>(p) = raw;
    }
}

}  // namespace fb

extern "C" {
int fbk_kv4_append(const fbx_kv4_cache& c, int type, const void* q, const void* k, const void* v, int64_t ldq,
                   int64_t ldkv, int T, int H, const int32_t* tok_seq, const int32_t* tok_pos, int rot, int neox,
                   const float* rcos, const float* rsin, int n_rope, int out_type, void* q_out, int64_t ldq_out,
                   void* k_out, void* v_out, int64_t ldkv_out, cudaStream_t st);
size_t fbk_kv4_attention_workspace(int T, int H, int HKV, int D, int max_keys);
int fbk_kv4_attention(const fbx_kv4_cache& c, int type, const void* q, int64_t ldq, int T, int H, const int32_t* tok_seq,
                      const int32_t* tok_pos, int max_keys, float scale, float softcap, int window, void* out, int64_t ldo,
                      void* ws, cudaStream_t st);
int fbk_attention_packed(int type, const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv, int n_rows,
                         const int32_t* cu, int B, int H, int HKV, int D, float scale, float softcap, int window,
                         void* out, int64_t ldo, cudaStream_t st);
}
