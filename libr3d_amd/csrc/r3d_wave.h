/* r3d_wave.h -- sums and maxima over the lanes of a wave by moves between registers (row rotations, shifts
 * and broadcasts of gfx9's vector unit): a step takes two or three instructions, where an exchange by way
 * of LDS has the lanes wait some 60 cycles for each. */
#ifndef R3D_WAVE_H
#define R3D_WAVE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

/* The largest over each 16 lanes, by rotations of the register (no lane waits for LDS). */
__device__ __forceinline__ float r3d_max16(float v) {
#define R3D_ROTATE(N_) \
    v = __builtin_fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x120 + N_, 15, 15, true)))
    R3D_ROTATE(8); R3D_ROTATE(4); R3D_ROTATE(2); R3D_ROTATE(1);
#undef R3D_ROTATE
    return v;
}

/* The sum over this lane and the ones before it in the wave, by row shifts and broadcasts. */
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t r3d_moved(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 15, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 15, false);
    return (uint64_t)hi << 32 | lo;
}
template <class V>
__device__ __forceinline__ V r3d_scan16(V v) {                      /* within each 16 lanes */
#define R3D_STEP(CTRL_, ROWS_) v += __builtin_bit_cast(V, r3d_moved<CTRL_, ROWS_>(__builtin_bit_cast(uint64_t, v)))
    R3D_STEP(0x111, 15); R3D_STEP(0x112, 15); R3D_STEP(0x114, 15); R3D_STEP(0x118, 15);
    return v;
}
template <class V>
__device__ __forceinline__ V r3d_wave_scan(V v) {
    v = r3d_scan16(v);
    R3D_STEP(0x142, 10); R3D_STEP(0x143, 12);                       /* the 16 before, the 32 before */
#undef R3D_STEP
    return v;
}
/* Lane i's, i uniform. */
template <class V>
__device__ __forceinline__ V r3d_lane(V v, int i) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, i), hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), i);
    return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
}

/* The sum, or the largest, over all lanes of the wave, on every lane. */
__device__ __forceinline__ double r3d_wave_sum(double v) { return r3d_lane(r3d_wave_scan(v), 63); }
__device__ __forceinline__ uint32_t r3d_wave_max(uint32_t v) {
#define R3D_STEP(CTRL_, ROWS_) \
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL_, ROWS_, 15, false))
    R3D_STEP(0x111, 15); R3D_STEP(0x112, 15); R3D_STEP(0x114, 15); R3D_STEP(0x118, 15);
    R3D_STEP(0x142, 10); R3D_STEP(0x143, 12);
#undef R3D_STEP
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

#endif /* R3D_WAVE_H */
