// serving.hpp -- launchers of the kernels between the projections of many requests
// (kvcache.hip, paged_attention.hip), internal to libprism_hip.
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

// Scratch of an attention call (partial results of key ranges; 0: none).
size_t attention_scratch_bytes(const prism_kv_cache &cache, const prism_attention &a, uint32_t cus);
int launch_attention_paged(const prism_kv_cache &cache, const prism_attention &a, void *scratch, uint32_t cus, int *err,
                           hipStream_t s);

}  // namespace prism
