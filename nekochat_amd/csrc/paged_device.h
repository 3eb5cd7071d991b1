// Wave-level searches over a paged batch and the E4M3 conversions. All 64 lanes call each of these together.
#pragma once

#include "paged.h"

namespace neko_hip {

// The last of n >= 1 sequences whose start(s) <= x (0 if there is none), start being non-decreasing: 64 probes a
// step, so one load for up to 64 sequences and two for up to 4096.
template <typename F>
__device__ __forceinline__ int32_t wave_last(int32_t n, int32_t x, F&& start) {
    const int32_t lane = static_cast<int32_t>(threadIdx.x) & 63;
    int32_t lo = 0;
    while (n > 64) {
        const int32_t step = (n + 63) / 64;
        const int32_t at = lane * step;
        const bool le = at < n && start(lo + at) <= x;
        const int32_t hits = __popcll(__ballot(le));
        const int32_t skip = hits > 0 ? (hits - 1) * step : 0;
        lo += skip;
        n = n - skip < step ? n - skip : step;
    }
    const bool le = lane < n && start(lo + lane) <= x;
    const int32_t hits = __popcll(__ballot(le));
    return __builtin_amdgcn_readfirstlane(lo + (hits > 0 ? hits - 1 : 0));
}

// Two E4M3 codes, the low (HI = false) or high half of a dword, as f16: exact, NaN codes give NaN.
template <bool HI>
__device__ __forceinline__ half2v f16_of_fp8(uint32_t codes) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(codes), 1.0f, HI));
}

// 2^e for e within the normal range.
__device__ __forceinline__ float exp2i(int e) { return __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23); }

// Four values, times a power of two, as E4M3 codes: nearest, ties to even. What no scale brings to 448 (infinities,
// f32 values past 448 * 2^kScaleMax) and NaN are held as NaN. The product is exact but for results far below the
// smallest code.
__device__ __forceinline__ uint32_t fp8_of_f32(const float* x, float scale) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = x[i] * scale;
    uint32_t r = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false));
    r = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], static_cast<int>(r), true));
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (!(fabsf(y[i]) <= 448.0f)) r |= 0x7Fu << (8 * i);
    return r;
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto step = [&](uint32_t w) { v = v > w ? v : w; };
    step(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kDppQuadXor1, 0xF, 0xF, false)));
    step(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kDppQuadXor2, 0xF, 0xF, false)));
    step(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kDppRowHalfMirror, 0xF, 0xF, false)));
    step(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kDppRowMirror, 0xF, 0xF, false)));
    const uint32_t a = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 0));
    const uint32_t b = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 16));
    const uint32_t c = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 32));
    const uint32_t d = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 48));
    const uint32_t ab = a > b ? a : b, cd = c > d ? c : d;
    return ab > cd ? ab : cd;
}

}  // namespace neko_hip
