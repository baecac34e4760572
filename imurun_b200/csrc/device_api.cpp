// device_api.cpp — entry points on device buffers (include/fish/fish_kernels.h):
// the 4-bit cache and packed prompt attention. Argument checks; the kernels
// and their launches are in kernels/kv4.cu and kernels/attention_packed.cu.
#include <fish/fish_kernels.h>

#include <cuda_runtime.h>

#include <climits>
#include <initializer_list>

#include "kernels/kv4.cuh"

using namespace fb;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// arrays of 32-bit values; null passes
bool aligned4(std::initializer_list<const void*> ps) {
    uintptr_t all = 0;
    for (const void* p : ps) all |= reinterpret_cast<uintptr_t>(p);
    return (all & 3) == 0;
}
size_t type_bytes(int type) { return type == T_F32 ? 4 : type == T_F16 || type == T_BF16 ? 2 : 0; }
constexpr float kMost = 1e30f;
// what scores are multiplied by stays finite
bool scale_ok(float scale, float softcap) {
    return scale > 0.0f && scale <= kMost && (softcap == 0.0f || (softcap > 0.0f && softcap <= kMost && scale / softcap <= kMost && 1.0f / softcap <= kMost));
}
bool head_dim_ok(int D) { return D == 64 || D == 96 || D == 128; }

// a row stride that holds `width` values and keeps rows on 16-byte boundaries
bool stride_ok(int64_t ld, int64_t width, int type) {
    return ld >= width && ld <= ((int64_t)1 << 40) && (ld * (int64_t)type_bytes(type)) % 16 == 0;
}

// A buffer is memory that the current device can use as its own: a host array
// or another GPU's buffer would fault in the kernel. 0, -1 or a CUDA error. A
// look at a pointer takes 0.2 us, so of buffers that come in pairs (k and v, cos
// and sin) one is looked at.
int on_device(std::initializer_list<const void*> ps) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    for (const void* p : ps) {
        if (!p) continue;
        cudaPointerAttributes a{};
        e = cudaPointerGetAttributes(&a, p);
        if (e != cudaSuccess) return (int)e;
        if (a.type == cudaMemoryTypeManaged) continue;
        if (a.type != cudaMemoryTypeDevice || a.device != dev) return -1;
    }
    return 0;
}

bool cache_ok(const fbx_kv4_cache* c) {
    if (!c || !c->pool || !c->page_table || !aligned16(c->pool) || !aligned4({c->page_table, c->err})) return false;
    const size_t layer = fbx_kv4_layer_bytes(c->n_head_kv, c->head_dim);
    return layer && c->n_pages > 0 && c->table_stride > 0 && c->n_seqs > 0 && c->layer_offset >= 0 &&
           c->layer_offset % 16 == 0 && c->page_stride % 16 == 0 && c->page_stride - c->layer_offset >= (int64_t)layer;
}

}  // namespace

extern "C" {

FISH_API size_t fbx_kv4_layer_bytes(int n_head_kv, int head_dim) {
    if (n_head_kv <= 0 || n_head_kv > 65535) return 0;
    const size_t rec = head_dim == 128 ? Kv4Rec<128>::bytes : head_dim == 96 ? Kv4Rec<96>::bytes : head_dim == 64 ? Kv4Rec<64>::bytes : 0;
    return rec * (size_t)n_head_kv;
}

FISH_API int fbx_kv4_append(const fbx_kv4_cache* c, int type, const void* q, const void* k, const void* v, int64_t ldq,
                            int64_t ldkv, int T, int H, const int32_t* tok_seq, const int32_t* tok_pos, int rot, int neox,
                            const float* rope_cos, const float* rope_sin, int n_rope, int out_type, void* q_out,
                            int64_t ldq_out, void* k_out, void* v_out, int64_t ldkv_out, void* stream) {
    if (!cache_ok(c) || !type_bytes(type) || !type_bytes(out_type) || T < 0) return -1;
    if (T == 0) return 0;
    if (!k || !v || !tok_seq || !tok_pos) return -1;
    const int D = c->head_dim, HKV = c->n_head_kv;
    if ((q == nullptr) != (q_out == nullptr)) return -1;
    if (rot < 0 || rot > D || rot % 2 || (rot > 0 && (n_rope <= 0 || !rope_cos || !rope_sin))) return -1;
    if (rot == 0) {   // no tables, and so none to bound a position
        rope_cos = rope_sin = nullptr;
        n_rope = INT_MAX;
    }
    if (q && (H <= 0 || H > 65535 || !stride_ok(ldq, (int64_t)H * D, type) || !stride_ok(ldq_out, (int64_t)H * D, out_type)))
        return -1;
    if (!stride_ok(ldkv, (int64_t)HKV * D, type)) return -1;
    if ((k_out || v_out) && !stride_ok(ldkv_out, (int64_t)HKV * D, out_type)) return -1;
    for (const void* p : {q, k, v, (const void*)q_out, (const void*)k_out, (const void*)v_out})
        if (!aligned16(p)) return -1;
    if (!aligned4({tok_seq, tok_pos, rope_cos, rope_sin})) return -1;
    // in place means the same rows
    if (q && q == q_out && (type != out_type || ldq != ldq_out)) return -1;
    if ((k == k_out || v == v_out) && (type != out_type || ldkv != ldkv_out)) return -1;
    const int rc = on_device({c->pool, c->page_table, c->err, q, k, tok_pos, rope_cos, q_out, k_out ? k_out : v_out});
    if (rc) return rc;
    return fbk_kv4_append(*c, type, q, k, v, ldq, ldkv, T, H, tok_seq, tok_pos, rot, neox ? 1 : 0, rope_cos, rope_sin, n_rope,
                          out_type, q_out, ldq_out, k_out, v_out, ldkv_out, static_cast<cudaStream_t>(stream));
}

FISH_API size_t fbx_kv4_attention_workspace(int T, int H, int n_head_kv, int head_dim, int max_keys) {
    if (T <= 0 || n_head_kv <= 0 || H <= 0 || H % n_head_kv || !head_dim_ok(head_dim) || max_keys <= 0) return 0;
    return fbk_kv4_attention_workspace(T, H, n_head_kv, head_dim, max_keys);
}

FISH_API int fbx_kv4_attention(const fbx_kv4_cache* c, int type, const void* q, int64_t ldq, int T, int H,
                               const int32_t* tok_seq, const int32_t* tok_pos, int max_keys, float scale, float softcap,
                               int window, void* out, int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
    if (!cache_ok(c) || !type_bytes(type) || T < 0 || T > 65535 || max_keys <= 0) return -1;
    if (T == 0) return 0;
    if (!q || !out || !tok_seq || !tok_pos) return -1;
    const int D = c->head_dim, HKV = c->n_head_kv;
    if (H <= 0 || H > 65535 || H % HKV || !scale_ok(scale, softcap) || window < 0) return -1;
    if (!stride_ok(ldq, (int64_t)H * D, type) || !stride_ok(ldo, (int64_t)H * D, type)) return -1;
    if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || !aligned4({tok_seq, tok_pos})) return -1;
    const size_t need = fbk_kv4_attention_workspace(T, H, HKV, D, max_keys);
    if (need && (!workspace || workspace_bytes < need)) return -1;
    const int rc = on_device({c->pool, c->page_table, c->err, q, tok_pos, out, need ? workspace : nullptr});
    if (rc) return rc;
    return fbk_kv4_attention(*c, type, q, ldq, T, H, tok_seq, tok_pos, max_keys, scale, softcap, window, out, ldo, workspace,
                             static_cast<cudaStream_t>(stream));
}

FISH_API int fbx_attention_packed(int type, const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv,
                                  int n_rows, const int32_t* cu_seqlens, int n_seqs, int H, int HKV, int D, float scale,
                                  float softcap, int window, void* out, int64_t ldo, void* stream) {
    if ((type != T_F16 && type != T_BF16) || n_rows < 0 || n_seqs <= 0 || n_seqs > (1 << 20) || n_rows > (1 << 30)) return -1;
    if (n_rows == 0) return 0;
    if (!q || !k || !v || !out || !cu_seqlens) return -1;
    if (!head_dim_ok(D) || HKV <= 0 || H <= 0 || H % HKV || H > 65535 || H / HKV > 128 || !scale_ok(scale, softcap) || window < 0)
        return -1;
    if (!stride_ok(ldq, (int64_t)H * D, type) || !stride_ok(ldkv, (int64_t)HKV * D, type) ||
        !stride_ok(ldo, (int64_t)H * D, type))
        return -1;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned4({cu_seqlens})) return -1;
    const int rc = on_device({q, k, cu_seqlens, out});
    if (rc) return rc;
    return fbk_attention_packed(type, q, ldq, k, v, ldkv, n_rows, cu_seqlens, n_seqs, H, HKV, D, scale, softcap, window, out,
                                ldo, static_cast<cudaStream_t>(stream));
}

}
