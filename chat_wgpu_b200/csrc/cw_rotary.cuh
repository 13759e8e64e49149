// cw_rotary.cuh -- what the kernels that rotate rows share: vectors of a type's elements
// and the sines of a position.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "cw_device.cuh"

namespace cw {

template <int BYTES> struct VecOf;
template <> struct VecOf<16> { typedef uint4 type; };
template <> struct VecOf<8> { typedef uint2 type; };
template <> struct VecOf<4> { typedef uint32_t type; };
template <> struct VecOf<2> { typedef uint16_t type; };

__device__ __forceinline__ float rp_f32(float x) { return x; }
__device__ __forceinline__ float rp_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float rp_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void rp_set(float* d, float x) { *d = x; }
__device__ __forceinline__ void rp_set(__half* d, float x) { *d = __float2half_rn(x); }
__device__ __forceinline__ void rp_set(__nv_bfloat16* d, float x) { *d = __float2bfloat16_rn(x); }

// Cosines and sines, times amp, of the N pairs whose turns per position are steps[0..N).
// The angle is formed in turns as 64-bit fixed point: position * step wraps modulo one turn
// exactly, so the f32 that goes to sincospif is within half a turn at any position.
template <typename T, int N>
__device__ __forceinline__ void rotary_sines(const unsigned long long* steps, long long pos,
                                             float amp, float* cs, float* sn) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        const long long ph = (long long)((unsigned long long)pos * steps[i]);
        // 16-bit values: within half a turn the fast functions are off by 2^-21
        if (sizeof(T) == 2) __sincosf((float)ph * 0x1.921fb6p-62f, &sn[i], &cs[i]);
        else sincospif((float)ph * 0x1p-63f, &sn[i], &cs[i]);
        sn[i] *= amp;
        cs[i] *= amp;
    }
}

}  // namespace cw
