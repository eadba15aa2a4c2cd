// serving.hpp -- launchers of the kernels between the projections of many requests
// (kvcache.hip, kvcache4.hip, paged_attention.hip, paged_attention4.hip) and behind their head
// (logprobs.hip), internal to libprism_hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "prism_hip.h"

namespace prism {

// Scratch of a plan of `requests` requests.
size_t plan_scratch_bytes(uint32_t requests);
int launch_kv_plan(const prism_kv_plan &p, void *scratch, int *err, hipStream_t s);

// The rotation of a prism_hip_rope: freq[dims / 2] on the device.
struct Rotation {
    const double *freq = nullptr;
    uint32_t dims = 0;  // 0: none
    int interleaved = 0;
    double magnitude = 1.0;
};
// Rows [tokens][heads][head_dim] of one tensor to rotate (x -> out; norm may be null).
struct RopeRows {
    const void *x = nullptr;
    void *out = nullptr;
    uint64_t x_stride = 0, out_stride = 0;
    uint32_t heads = 0;
    const float *norm = nullptr;
};
// One launch rotates both (b.heads may be 0).
int launch_rope(int dtype, const Rotation &rot, const RopeRows &a, const RopeRows &b, const int32_t *positions,
                uint32_t tokens, uint32_t head_dim, float eps, int *err, hipStream_t s);
int launch_kv_append(const prism_kv_cache &cache, int dtype, const void *k, uint64_t k_stride, const void *v,
                     uint64_t v_stride, const int32_t *slots, uint32_t tokens, int *err, hipStream_t s);
// The same into a cache of 4 bits a value (kvcache4.hip).
int launch_kv_append4(const prism_kv_cache &cache, int dtype, const void *k, uint64_t k_stride, const void *v,
                      uint64_t v_stride, const int32_t *slots, uint32_t tokens, int *err, hipStream_t s);
// Rotated q into memory, rotated k and v into a cache of 4 bits a value, in one launch; dims multiples of 8.
int launch_qkv_append4(const prism_kv_cache &cache, int dtype, const Rotation &rot, const RopeRows &q, const RopeRows &k, const void *v,
                       uint64_t v_stride, const int32_t *positions, const int32_t *slots, uint32_t tokens, float eps, int *err, hipStream_t s);
// Slots of a cache of any format as rows (k or v may be null).
int launch_kv_read(const prism_kv_cache &cache, int dtype, const int32_t *slots, uint32_t tokens, void *k, uint64_t k_stride,
                   void *v, uint64_t v_stride, int *err, hipStream_t s);

// Scratch of an attention call (partial results of key ranges; 0: none).
size_t attention_scratch_bytes(const prism_kv_cache &cache, const prism_attention &a, uint32_t cus);
int launch_attention_paged(const prism_kv_cache &cache, const prism_attention &a, void *scratch, uint32_t cus, int *err,
                           hipStream_t s);
// The same over a cache of 4 bits a value (paged_attention4.hip).
size_t attention4_scratch_bytes(const prism_kv_cache &cache, const prism_attention &a, uint32_t cus);
int launch_attention4_paged(const prism_kv_cache &cache, const prism_attention &a, void *scratch, uint32_t cus, int *err,
                            hipStream_t s);

// Log probabilities of rows of logits (logprobs.hip); scratch of rows split over workgroups (0: none).
size_t logprobs_scratch_bytes(const prism_logprobs &call, uint32_t cus);
int launch_logprobs(const prism_logprobs &call, void *scratch, uint32_t cus, int *err, hipStream_t s);

}  // namespace prism
