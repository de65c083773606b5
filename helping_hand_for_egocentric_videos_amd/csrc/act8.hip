// Activation checkpoints in 8 bits: what a backward pass needs of a forward activation u, kept as e4m3 values q with one scale s = 2^k for
// every 128 consecutive channels of a row, u ~ q * s.
//
//   forward:   a = act(u) from the exact u;  k = the smallest whole number with max|u| <= 448 * 2^k over the 128 channels (448 = 1.75 * 2^8 is
//              the largest e4m3 value; k is held in [-117, 120], and is 0 where all are zero);  q = u / s rounded to nearest, ties to even.
//              A power of two, because then u / s and q * s are exact in fp32, and q * s (4 significant bits) is exact in bf16 too: the matrix core
//              takes a checkpoint without a second rounding (gemm_tn8.hip), and the only error is e4m3's own half step, 2^-4 of the value
//              (2^-10 of s below 2^-6 of s).  k >= -117 keeps the smallest step, 2^(k - 9), a normal number.  At the other end of the range |u| from 1.9375 * 2^127
//              (3.29e38) on rounds to 2^128, the one q * s that fp32 and bf16 do not have: it is read back as infinity, as bf16 itself would round most of these.
//              Infinities and NaN do not count for the scale; both are stored as e4m3's NaN, so that a gradient that uses them shows it.
//   backward:  v = q * s;  du = da * act'(v), and on request act(v), the operand of the next product's weight gradient.
//
// Both are bound by HBM: a lane takes 8 channels (16 B of bf16), 16 lanes share a scale, one exchange over them.  32 776 x 4096 bf16 (QuickGELU): forward 112 us = 6.0
// TB/s, backward 106-107 us = 6.3 TB/s with outputs past the caches (a copy of 2 GiB: 4.9 TB/s).  A row that no 16 bytes divide is read and written in the same pieces, the
// last one moved back to end with the row (24 640 x 767: 20.7 us, one element at a time 52.7).
#include "common.h"

#define ACT8_GROUP 128

// sigmoid(1.702 v) on the hardware's exp2 and reciprocal (a unit in the last place each; a result below 2^-126, v < -51.3, is zero).  With expf and a division both
// passes over 32 776 x 4096 bf16 were bound by their arithmetic (143 and 135 us).
__device__ __forceinline__ float sigmoid1702(float v) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * (-1.702f * 1.4426950408889634f))); }
__device__ __forceinline__ float act_value(float v, int act) {
    if (act == HH_ACT_QUICKGELU) return v * sigmoid1702(v);
    if (act == HH_ACT_RELU) return v < 0.f ? 0.f : v;             // (keeps NaN)
    return v;
}
__device__ __forceinline__ float act_slope(float v, int act) {
    if (act == HH_ACT_QUICKGELU) {
        // s is 0 below -52 and 1 above 11 (to fp32): v no longer counts there, and 1.702 v, which is infinite from 2^127 / 0.851 on, stays finite.  s keeps NaN.
        const float s = sigmoid1702(v);
        return s * (1.f + 1.702f * __builtin_amdgcn_fmed3f(v, -128.f, 128.f) * (1.f - s));
    }
    if (act == HH_ACT_RELU) return v > 0.f ? 1.f : v <= 0.f ? 0.f : v;      // (keeps NaN)
    return 1.f;
}

// act(v) of a checkpoint's value, which is infinite where a finite activation was rounded up to 2^128: QuickGELU of minus infinity is 0, not infinity * 0
__device__ __forceinline__ float act_again(float v, int act) {
    if (act == HH_ACT_QUICKGELU) return fmaxf(v, -3.402823466e38f) * sigmoid1702(v);
    return act_value(v, act);
}

template <typename T, bool NT>
__device__ __forceinline__ void load8(const T* p, bool whole, int n, float (&v)[8]) {
    if (whole) {
        if constexpr (sizeof(T) == 4) {
            const f32x4 a = NT ? __builtin_nontemporal_load((const f32x4_any*)p) : *(const f32x4_any*)p;
            const f32x4 b = NT ? __builtin_nontemporal_load((const f32x4_any*)(p + 4)) : *(const f32x4_any*)(p + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
        } else {
            const u32x4 t = NT ? __builtin_nontemporal_load((const u32x4_any*)p) : *(const u32x4_any*)p;
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[2 * j] = bf16_lo_to_f32(t[j]); v[2 * j + 1] = bf16_hi_to_f32(t[j]); }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.f;
    }
}
template <typename T, bool NT>
__device__ __forceinline__ void store8(T* p, bool whole, int n, const float (&v)[8]) {
    if (whole) {
        if constexpr (sizeof(T) == 4) {
            const f32x4_any a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
            f32x4_any* o = (f32x4_any*)p;
            if (NT) { __builtin_nontemporal_store(a, o); __builtin_nontemporal_store(b, (f32x4_any*)(p + 4)); } else { *o = a; *(f32x4_any*)(p + 4) = b; }
        } else {
            const u32x4_any t = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
            u32x4_any* o = (u32x4_any*)p;
            if (NT) __builtin_nontemporal_store(t, o); else *o = t;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) p[j] = (T)v[j];
    }
}

__device__ __forceinline__ float pow2(int k) { return __uint_as_float((unsigned)(k + 127) << 23); }

// The group of 128 channels that 16 lanes share, and this lane's 8 of them.  Rows of whole groups are one long list (log_p < 0): no division.  Otherwise a
// workgroup's 16 groups are those of 16 >> log_p rows, or, with log_p = 4, a part of one row.
struct Act8Place { int64_t group, at; int left; };
__device__ __forceinline__ Act8Place act8_place(int per_row, int cols, int log_p, int parts, int64_t rows, bool* on) {
    const int t = threadIdx.x >> 4, c0 = (threadIdx.x & 15) * 8;
    Act8Place q;
    if (log_p < 0) {
        q.group = (int64_t)blockIdx.x * 16 + t;
        *on = q.group < rows * per_row;
        q.at = q.group * ACT8_GROUP + c0;
        q.left = ACT8_GROUP - c0;
        return q;
    }
    const unsigned block = blockIdx.x / (unsigned)parts, part = blockIdx.x % (unsigned)parts;
    const int64_t row = (int64_t)block * (16 >> log_p) + (t >> log_p);
    const int gi = (int)part * 16 + (t & ((1 << log_p) - 1));
    *on = row < rows && gi < per_row;
    q.group = row * per_row + gi;
    q.at = row * cols + gi * ACT8_GROUP + c0;
    q.left = cols - gi * ACT8_GROUP - c0;                            // may be <= 0
    // the piece in which the row ends is moved back to be whole, inside its group: what it shares with the piece before is worked out twice, to the same values
    if (q.left > 0 && q.left < 8 && c0 > 0) { q.at -= 8 - q.left; q.left = 8; }
    return q;
}

template <typename T, bool NT>
__global__ __launch_bounds__(256) void act8_fwd_kernel(const T* __restrict__ u, T* __restrict__ a, unsigned char* __restrict__ q, float* __restrict__ scale, int64_t rows, int per_row,
                                                       int cols, int log_p, int parts, int act) {
    bool on;
    const Act8Place place = act8_place(per_row, cols, log_p, parts, rows, &on);
    if (!on) return;                                                     // (16 lanes at a time: the exchange below stays inside them)
    const int64_t g = place.group, at = place.at;
    const int n = place.left;
    const bool whole = n >= 8;
    float v[8];
    load8<T, NT>(u + at, whole, n, v);
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float m = fabsf(v[j]);
        top = fmaxf(top, m <= 3.402823466e38f ? m : 0.f);                // (false for NaN and infinity)
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    int k = 0;
    if (top > 0.f) {
        const unsigned b = __float_as_uint(top);
        k = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u);     // 1.75 is the mantissa 0x600000; subnormals land below the clamp
        k = k < -117 ? -117 : k > 120 ? 120 : k;
    }
    if ((threadIdx.x & 15) == 0) scale[g] = pow2(k);
    const float inv = pow2(-k);
    unsigned w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * inv, v[4 * h + 1] * inv, 0, false);
        w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * inv, v[4 * h + 3] * inv, w[h], true);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (!(fabsf(v[4 * h + j]) <= 3.402823466e38f)) w[h] |= 0x7fu << (8 * j);
    }
    if (whole) {
        const u32x2_any t = {w[0], w[1]};
        u32x2_any* o = (u32x2_any*)(q + at);
        if (NT) __builtin_nontemporal_store(t, o); else *o = t;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) q[at + j] = (unsigned char)(w[j >> 2] >> (8 * (j & 3)));
    }
    if (a != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = act_value(v[j], act);
        store8<T, NT>(a + at, whole, n, v);
    }
}

template <typename T, bool NT>
__global__ __launch_bounds__(256) void act8_bwd_kernel(const unsigned char* __restrict__ q, const float* __restrict__ scale, const T* __restrict__ da, T* __restrict__ du, T* __restrict__ a,
                                                       int64_t rows, int per_row, int cols, int log_p, int parts, int act) {
    bool on;
    const Act8Place place = act8_place(per_row, cols, log_p, parts, rows, &on);
    if (!on) return;
    const int64_t g = place.group, at = place.at;
    const int n = place.left;
    const bool whole = n >= 8;
    unsigned w[2] = {0u, 0u};
    if (whole) {
        const u32x2 t = NT ? __builtin_nontemporal_load((const u32x2_any*)(q + at)) : *(const u32x2_any*)(q + at);
        w[0] = t[0]; w[1] = t[1];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) w[j >> 2] |= (unsigned)q[at + j] << (8 * (j & 3));
    }
    const float s = scale[g];
    float v[8], d[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[h], true);
        v[4 * h] = lo[0] * s; v[4 * h + 1] = lo[1] * s;
        v[4 * h + 2] = hi[0] * s; v[4 * h + 3] = hi[1] * s;
    }
    load8<T, NT>(da + at, whole, n, d);
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] *= act_slope(v[j], act);
    store8<T, NT>(du + at, whole, n, d);
    if (a != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = act_again(v[j], act);
        store8<T, NT>(a + at, whole, n, v);
    }
}

struct Act8Grid { int64_t blocks; int log_p, parts; };
static Act8Grid act8_grid(int64_t rows, int cols) {
    const int per_row = (cols + ACT8_GROUP - 1) / ACT8_GROUP;
    Act8Grid g = {0, -1, 1};
    if (cols % ACT8_GROUP == 0) {
        g.blocks = (rows * per_row + 15) / 16;
        return g;
    }
    g.log_p = 0;
    while (g.log_p < 4 && (1 << g.log_p) < per_row) ++g.log_p;
    g.parts = (per_row + 15) / 16;
    const int64_t at_once = 16 >> g.log_p;
    g.blocks = (rows + at_once - 1) / at_once * g.parts;
    return g;
}
static bool act8_ok(int act) { return act == HH_ACT_NONE || act == HH_ACT_QUICKGELU || act == HH_ACT_RELU; }

extern "C" int hh_act8_fwd(const void* u, int u_dtype, void* a, void* q, float* scale, int64_t rows, int cols, int act, hh_stream_t stream) {
    HH_REQUIRE(rows >= 0 && cols > 0, HH_ERR_SHAPE, "hh_act8_fwd: rows=%lld cols=%d", (long long)rows, cols);
    HH_REQUIRE(u_dtype == HH_F32 || u_dtype == HH_BF16, HH_ERR_DTYPE, "hh_act8_fwd: bad dtype");
    HH_REQUIRE(act8_ok(act), HH_ERR_UNSUPPORTED, "hh_act8_fwd: unknown activation %d", act);
    const int per_row = (cols + ACT8_GROUP - 1) / ACT8_GROUP;
    HH_REQUIRE(rows < (1ll << 40) && hh_grid_fits(act8_grid(rows, cols).blocks, 256), HH_ERR_SHAPE, "hh_act8_fwd: too many rows for a launch (rows=%lld cols=%d)", (long long)rows, cols);
    const Act8Grid g = act8_grid(rows, cols);
    const int64_t blocks = g.blocks;
    if (rows == 0) return HH_OK;
    HH_REQUIRE(u != nullptr && q != nullptr && scale != nullptr, HH_ERR_ALIGN, "hh_act8_fwd: NULL pointer");
    const bool f32 = u_dtype == HH_F32, nt = rows * cols * (1 + (a ? (f32 ? 4 : 2) : 0)) > HH_STREAM_BYTES;
#define AF(T, N) hipLaunchKernelGGL((act8_fwd_kernel<T, N>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, (const T*)u, (T*)a, (unsigned char*)q, scale, rows, per_row, cols, g.log_p, g.parts, act)
    if (f32) { if (nt) AF(float, true); else AF(float, false); }
    else { if (nt) AF(bf16_t, true); else AF(bf16_t, false); }
#undef AF
    return hh_check_launch("hh_act8_fwd");
}

extern "C" int hh_act8_bwd(const void* q, const float* scale, const void* da, void* du, void* a, int dtype, int64_t rows, int cols, int act, hh_stream_t stream) {
    HH_REQUIRE(rows >= 0 && cols > 0, HH_ERR_SHAPE, "hh_act8_bwd: rows=%lld cols=%d", (long long)rows, cols);
    HH_REQUIRE(dtype == HH_F32 || dtype == HH_BF16, HH_ERR_DTYPE, "hh_act8_bwd: bad dtype");
    HH_REQUIRE(act8_ok(act), HH_ERR_UNSUPPORTED, "hh_act8_bwd: unknown activation %d", act);
    const int per_row = (cols + ACT8_GROUP - 1) / ACT8_GROUP;
    HH_REQUIRE(rows < (1ll << 40) && hh_grid_fits(act8_grid(rows, cols).blocks, 256), HH_ERR_SHAPE, "hh_act8_bwd: too many rows for a launch (rows=%lld cols=%d)", (long long)rows, cols);
    const Act8Grid g = act8_grid(rows, cols);
    const int64_t blocks = g.blocks;
    if (rows == 0) return HH_OK;
    HH_REQUIRE(q != nullptr && scale != nullptr && da != nullptr && du != nullptr, HH_ERR_ALIGN, "hh_act8_bwd: NULL pointer");
    const bool f32 = dtype == HH_F32, nt = rows * cols * (f32 ? 4 : 2) * (a ? 2 : 1) > HH_STREAM_BYTES;
#define AB(T, N) hipLaunchKernelGGL((act8_bwd_kernel<T, N>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, (const unsigned char*)q, scale, (const T*)da, (T*)du, (T*)a, rows, per_row, cols, g.log_p, g.parts, act)
    if (f32) { if (nt) AB(float, true); else AB(float, false); }
    else { if (nt) AB(bf16_t, true); else AB(bf16_t, false); }
#undef AB
    return hh_check_launch("hh_act8_bwd");
}
