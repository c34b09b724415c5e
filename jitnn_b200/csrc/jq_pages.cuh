// What the operators of paged decoding share: element types, the handles, and how a row of a batch finds its sequence.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "jq_common.cuh"

namespace jq {

constexpr int BOX_KEYS = 128;  // of a tensor map's box, where a page has as many

inline int elem_bytes(int elem) { return elem == JQ_ELEM_F32 ? 4 : 2; }
inline bool elem_ok(int elem) { return elem == JQ_ELEM_F32 || elem == JQ_ELEM_F16 || elem == JQ_ELEM_BF16; }
inline const char* elem_name(int elem) { return elem == JQ_ELEM_F32 ? "FP32" : (elem == JQ_ELEM_F16 ? "FP16" : (elem == JQ_ELEM_BF16 ? "BF16" : "?")); }

// Codes of the status word (jq_device_status) for what only the device sees.
constexpr int STATUS_PAGE = 96;      // a page id, or a position, that the cache or the table of pages does not have
constexpr int STATUS_POSITION = 97;  // a position that the table of rotations does not have
constexpr int STATUS_TOKEN = 98;     // a drafted token outside the vocabulary

__device__ __forceinline__ void note_status(int* status, int code) {
    *reinterpret_cast<volatile int*>(status) = code;  // (page-locked host memory; of several codes any one will do)
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The rows of a call and the sequences they belong to: rows starts[s] .. starts[s + 1] - 1 are the newest of sequence s, which has lengths[s] keys of its own once they
// are appended, on the pages tables[s][0 ..]. In front of them all sequences see the prefix_length keys on the pages prefix[0 ..].
struct Batch {
    const int* tables;
    int64_t table_stride;
    int table_width;
    const int* starts;
    const int* lengths;
    int sequences;
    const int* prefix;
    int prefix_length;
    int tokens;
};

}  // namespace jq

// The handles of the C ABI.
struct jq_rope {
    uint32_t magic;
    int device;
    int dim;         // rotated elements of a head
    int interleaved;
    int64_t positions;
    float2* table;   // [positions][dim / 2]: cosine and sine, times the magnitude
};
struct jq_pages {
    uint32_t magic;
    int device;
    int elem;
    int page_size, kv_heads, head_dim;
    int64_t pages;
    void *k, *v;     // [pages][kv_heads][page_size][head_dim], the caller's
    CUtensorMap k_map, v_map;  // of 16-bit pages with heads of 64 or 128: boxes of 64 elements of up to 128 keys
};
#define JQ_ROPE_MAGIC 0x4a51524fu
#define JQ_PAGES_MAGIC 0x4a515047u

namespace jq {
int check_rope(const jq_rope* r, const char* who);
int check_pages(const jq_pages* p, const char* who);
int check_batch(const jq_pages* p, const Batch& b, const char* who);
}  // namespace jq
