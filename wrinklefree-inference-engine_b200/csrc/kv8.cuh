// How rows of keys and values are kept in an int8 pool.
#pragma once
#include "common.cuh"

namespace wf {

// per-(token, head) symmetric int8 quantisation, the reference's arithmetic (kv_cache.py:198-218) at token granularity:
// scale = 127 / absmax (absmax < 1e-6 -> 1), code = clamp(round(x * scale), -127, 127), stored dequant scale = absmax / 127
__device__ __forceinline__ float kv8_inv(float& amax) {
    if (amax < 1e-6f) amax = 1.0f;
    return __fdiv_rn(127.0f, amax);
}
__device__ __forceinline__ int kv8_code(float x, float inv) { return (int)fminf(fmaxf(rintf(__fmul_rn(x, inv)), -127.f), 127.f); }
__device__ __forceinline__ uint8_t kv8_store(float x, float inv) { return (uint8_t)(kv8_code(x, inv) + 128); }   // offset binary
__device__ __forceinline__ float kv8_scale(float amax) { return __fdiv_rn(amax, 127.0f); }

}  // namespace wf
