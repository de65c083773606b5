// The end of a residual block in one pass over its rows, and its gradients:
//     p = post(y)  (a norm, or y itself),   x_new = res_scale * x + g o p,   h = pre(x_new)  (the next block's norm, or nothing)
// where a norm is gamma o (v - mean) * rstd + beta (LayerNorm) or gamma o v * rrms (+ beta), and the gate g is 1, a scalar, a row over the
// channels, or such a row for each group of consecutive rows, as it is or through tanh (the tanh gate of model/LaviLa.py:305-390 is the scalar one).
// Statistics are two-pass and in fp32, from the fp32 x_new before it is rounded to its storage type.
//
// Backward, from x_new, y and the gradients dx_new, dh (statistics are taken again: both rows are in registers anyway, and nothing has to be kept):
//     d = dx_new + pre'(dh),   dx = res_scale * d,   dgate = sum d o p (* 1 - tanh^2),   dy = post'(g o d),
//     n'(dn) = rstd * (k - mean(k) - xh * mean(k o xh)) with k = dn o gamma and xh the normed row   (no mean(k) term for root-mean-square norms).
// The gate's and post's gradients all come from two column sums over the rows of a gate group, S0 = sum d and S1 = sum d o xh:
//     dgate = (gamma o S1 + beta o S0) (* 1 - tanh^2),   dgamma += g o S1,   dbeta += g o S0,
// so that a lane keeps four sums for a channel (with dh o xh and dh of pre) and never needs p itself.  Every workgroup sums its rows in registers and leaves
// one row of partial sums, which a second launch adds in a fixed order (no atomics: equal inputs give equal bits).
//
// Layout: a row lies across the ceil(cols / 256) waves of a workgroup, 4 channels to a lane; the workgroup takes R rows at a time, so that the
// parameters are read once for them, R rows of loads are in flight, and one exchange through LDS (one barrier) serves the sums of R rows.  A wave per row, the
// obvious form, holds 16 channels of five sums in a lane at 1024 channels: 256 registers, one wave to a SIMD, 1168 us for the backward pass of 131 104 rows.
// Measured, both norms: forward 131 104 x 1024 (fp32 stream, bf16 branch) 268 us = 6.0 TB/s, bound by HBM; backward of it 472 us = 5.1 TB/s, near HBM's rate for two thirds
// reads; backward 12 320 x 768 bf16 24.5 us and 5.5 for the second launch over the same inputs again and again, 31.0 and 7.0 over a few first ones, 32-33 for both with three sets of
// inputs in turn; its arithmetic (VALU 82 % busy) is as long as the traffic.
#include "common.h"

struct Q4 { float v[4]; };

struct RnParams {
    const void* x; const void* y; void* x_new; void* h;
    const void* dx_new; const void* dh; void* dx; void* dy;
    const float* gate; const float* g1; const float* b1; const float* g2; const float* b2;
    float* part;                       // [4][blocks][cols]: dgamma / dbeta of post, of pre
    float* gate_part;                  // [units][cols], or [units] for a scalar gate
    int64_t rows, each;                // rows of one gate group (all of them without groups)
    int64_t chunks;                    // units of a group: unit j takes the rows j R .. j R + R - 1 and every chunks R-th behind them
    int64_t units, per_block;          // units in all, and of one workgroup
    int cols, gate_kind, gate_tanh, rms;
    int x_dt, y_dt, h_dt;
    float eps1, eps2, res_scale;
};

// Types: HH_F32, HH_BF16, or RN_ANY, read at run time -- the form for rows that take no wide accesses.
#define RN_ANY 2
template <int DT> __device__ __forceinline__ bool rn_f32(int dt) { return DT == RN_ANY ? dt == HH_F32 : DT == HH_F32; }
// a row's address (the same in all lanes, so that a load is a scalar base and the lane's offset)
template <int DT, typename T>
__device__ __forceinline__ T* rn_row(T* base, int dt, int64_t off) { return base + off * (rn_f32<DT>(dt) ? 4 : 2); }

// four channels as they lie in memory: 4 dwords of fp32, 2 of bf16; turned into fp32 only when all loads of a step have been issued (a conversion behind
// each load would wait for it).  Rows of any width and alignment (not VEC): the four in which the row ends are read whole, from up to three channels before, and
// shifted into place by rn_cvt; only a row of fewer than four is read one by one.
__device__ __forceinline__ int rn_behind(int c, int cols) { return c + 4 > cols && cols >= 4 ? c + 4 - cols : 0; }
template <bool VEC, int DT, bool NT = false>
__device__ __forceinline__ u32x4 rn_raw(const char* row, int dt, int c, int cols) {
    u32x4 r = {0u, 0u, 0u, 0u};
    if (VEC) {
        if (rn_f32<DT>(dt)) {
            const u32x4* at = (const u32x4*)(row + (unsigned)(c * 4));
            r = NT ? __builtin_nontemporal_load(at) : *at;
        } else {
            const u32x2* at = (const u32x2*)(row + (unsigned)(c * 2));
            const u32x2 t = NT ? __builtin_nontemporal_load(at) : *at;
            r[0] = t[0]; r[1] = t[1];
        }
    } else if (cols >= 4) {
        c -= rn_behind(c, cols);
        if (rn_f32<DT>(dt)) {
            const u32x4_any* at = (const u32x4_any*)(row + (unsigned)(c * 4));
            r = NT ? __builtin_nontemporal_load(at) : *at;
        } else {
            const u32x2_any* at = (const u32x2_any*)(row + (unsigned)(c * 2));
            const u32x2 t = NT ? __builtin_nontemporal_load(at) : *at;
            r[0] = t[0]; r[1] = t[1];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < cols) {
                if (rn_f32<DT>(dt)) r[j] = ((const unsigned*)row)[c + j];
                else r[j >> 1] |= (unsigned)((const unsigned short*)row)[c + j] << (16 * (j & 1));
            }
    }
    return r;
}
template <bool VEC, int DT>
__device__ __forceinline__ Q4 rn_cvt(const u32x4& r, int dt, int behind) {
    Q4 q;
    if (rn_f32<DT>(dt)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) q.v[j] = __uint_as_float(r[j]);
    } else {
        q.v[0] = bf16_lo_to_f32(r[0]); q.v[1] = bf16_hi_to_f32(r[0]);
        q.v[2] = bf16_lo_to_f32(r[1]); q.v[3] = bf16_hi_to_f32(r[1]);
    }
    if (!VEC && behind) {
        if (behind & 1) { q.v[0] = q.v[1]; q.v[1] = q.v[2]; q.v[2] = q.v[3]; q.v[3] = 0.f; }
        if (behind & 2) { q.v[0] = q.v[2]; q.v[1] = q.v[3]; q.v[2] = q.v[3] = 0.f; }
    }
    return q;
}
template <bool VEC>
__device__ __forceinline__ Q4 rn_param(const float* base, int64_t off, int c, int cols) {
    if (c >= cols) return Q4{{0.f, 0.f, 0.f, 0.f}};
    return rn_cvt<VEC, HH_F32>(rn_raw<VEC, HH_F32>((const char*)(base + off), HH_F32, c, cols), HH_F32, rn_behind(c, cols));
}

template <bool VEC, bool NT, int DT>
__device__ __forceinline__ void rn_store(const Q4& q, char* row, int dt, int c, int cols) {
    if (VEC) {
        if (rn_f32<DT>(dt)) {
            const f32x4 t = {q.v[0], q.v[1], q.v[2], q.v[3]};
            f32x4* o = (f32x4*)(row + (unsigned)(c * 4));
            if (NT) __builtin_nontemporal_store(t, o); else *o = t;
        } else {
            const u32x2 t = {pack_bf16(q.v[0], q.v[1]), pack_bf16(q.v[2], q.v[3])};
            u32x2* o = (u32x2*)(row + (unsigned)(c * 2));
            if (NT) __builtin_nontemporal_store(t, o); else *o = t;
        }
    } else if (c + 4 <= cols) {
        if (rn_f32<DT>(dt)) {
            const f32x4_any t = {q.v[0], q.v[1], q.v[2], q.v[3]};
            f32x4_any* o = (f32x4_any*)(row + (unsigned)(c * 4));
            if (NT) __builtin_nontemporal_store(t, o); else *o = t;
        } else {
            const u32x2_any t = {pack_bf16(q.v[0], q.v[1]), pack_bf16(q.v[2], q.v[3])};
            u32x2_any* o = (u32x2_any*)(row + (unsigned)(c * 2));
            if (NT) __builtin_nontemporal_store(t, o); else *o = t;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (c + j < cols) {
                if (rn_f32<DT>(dt)) ((float*)row)[c + j] = q.v[j];
                else ((bf16_t*)row)[c + j] = (bf16_t)q.v[j];
            }
    }
}
template <bool VEC>
__device__ __forceinline__ void rn_put(const Q4& q, float* row, int c, int cols) {
    if (c < cols) rn_store<VEC, false, HH_F32>(q, (char*)row, HH_F32, c, cols);
}

__device__ __forceinline__ float add_swapped32(float a, float b) {     // lanes 0..31: a over both halves, lanes 32..63: b
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_swapped16(float a, float b) {     // even rows of 16 lanes: a over a pair of rows, odd rows: b
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float add_row16(float v) {                  // sum over the 16 lanes of a row, in every lane of it (row rotations)
    return add_dpp<0x121>(add_dpp<0x122>(add_dpp<0x124>(add_dpp<0x128>(v))));
}

// N values (1, 2, 4 or 8) summed over the workgroup, in every lane.  A wave halves the number of values that a lane holds with the number of lanes that hold a
// value (8 values: 20 instructions instead of 48 exchanges), the waves meet in LDS.  `turn` alternates between two buffers: a wave writes a buffer again
// only behind the barrier of the sums in between, which every wave passes after it has read.  Places of waves that there are not hold zeros (four are read
// at once).
struct RnRed { __attribute__((aligned(16))) float buf[2][16 * 8]; };
__device__ __forceinline__ void rn_clear(RnRed& red) {
    for (int i = threadIdx.x; i < 2 * 16 * 8; i += blockDim.x) red.buf[0][i] = 0.f;
    __syncthreads();
}
template <int N>
__device__ __forceinline__ void block_sums(float (&s)[N], RnRed& red, int& turn, int waves) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float* buf = red.buf[turn];
    turn ^= 1;
    if constexpr (N >= 4) {
        float t[N / 2], u[N / 4];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) t[i] = add_swapped32(s[i], s[i + N / 2]);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) u[i] = add_row16(add_swapped16(t[i], t[i + N / 4]));
        if ((lane & 15) == 0)
#pragma unroll
            for (int i = 0; i < N / 4; ++i) buf[wave * 8 + (lane >> 4) * (N / 4) + i] = u[i];
    } else if constexpr (N == 2) {
        float t = add_swapped32(s[0], s[1]);
        t = add_row16(add_swapped16(t, t));
        if ((lane & 31) == 0) buf[wave * 8 + (lane >> 5)] = t;
    } else {
        float t = add_swapped32(s[0], s[0]);
        t = add_row16(add_swapped16(t, t));
        if (lane == 0) buf[wave * 8] = t;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.f;
    for (int w = 0; w < waves; w += 4) {
        f32x4 a[4], b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            a[k] = *(const f32x4*)(buf + (w + k) * 8);
            if constexpr (N == 8) b[k] = *(const f32x4*)(buf + (w + k) * 8 + 4);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += i < 4 ? (a[0][i & 3] + a[1][i & 3]) + (a[2][i & 3] + a[3][i & 3]) : (b[0][i & 3] + b[1][i & 3]) + (b[2][i & 3] + b[3][i & 3]);
    }
}

// sum of a lane's four channels.  KNOWN: channels behind the row's end hold zeros already
template <bool KNOWN>
__device__ __forceinline__ float rn_sum4(const Q4& q, int c, int cols) {
    if (KNOWN) return (q.v[0] + q.v[1]) + (q.v[2] + q.v[3]);
    return ((c < cols ? q.v[0] : 0.f) + (c + 1 < cols ? q.v[1] : 0.f)) + ((c + 2 < cols ? q.v[2] : 0.f) + (c + 3 < cols ? q.v[3] : 0.f));
}

// mean and reciprocal standard deviation (or root mean square, with mean 0) of N rows; two passes
template <bool VEC, bool KNOWN, int N>
__device__ __forceinline__ void rn_stats(const Q4 (&v)[N], int c, int cols, float inv, int rms, const float (&eps)[N], RnRed& red, int& turn, int waves, float (&mean)[N], float (&rstd)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) mean[i] = 0.f;
    if (!rms) {
#pragma unroll
        for (int i = 0; i < N; ++i) mean[i] = rn_sum4<KNOWN>(v[i], c, cols);
        block_sums<N>(mean, red, turn, waves);
#pragma unroll
        for (int i = 0; i < N; ++i) mean[i] *= inv;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        Q4 q;
#pragma unroll
        for (int j = 0; j < 4; ++j) { const float d = v[i].v[j] - mean[i]; q.v[j] = d * d; }
        rstd[i] = VEC ? (c < cols ? rn_sum4<true>(q, c, cols) : 0.f) : rn_sum4<false>(q, c, cols);
    }
    block_sums<N>(rstd, red, turn, waves);
#pragma unroll
    for (int i = 0; i < N; ++i) rstd[i] = rsqrtf(rstd[i] * inv + eps[i]);
}

template <bool VEC>
__device__ __forceinline__ Q4 rn_gate(const RnParams& p, int64_t group, int c) {
    Q4 g = {{1.f, 1.f, 1.f, 1.f}};
    if (p.gate_kind == HH_GATE_NONE) return g;
    if (p.gate_kind == HH_GATE_SCALAR) {
#pragma unroll
        for (int j = 0; j < 4; ++j) g.v[j] = p.gate[0];
    } else {
        g = rn_param<VEC>(p.gate, p.gate_kind == HH_GATE_GROUP ? group * p.cols : 0, c, p.cols);
    }
    if (p.gate_tanh)
#pragma unroll
        for (int j = 0; j < 4; ++j) g.v[j] = tanhf(g.v[j]);
    return g;
}

template <int R, bool VEC, bool NT, int XT, int YT, int HT>
__global__ __launch_bounds__(1024) void resnorm_fwd_kernel(RnParams p) {
    __shared__ RnRed red;
    const int waves = blockDim.x >> 6, c = threadIdx.x * 4, behind = rn_behind(c, p.cols);
    const bool on = c < p.cols;
    const float inv = 1.f / (float)p.cols;
    const Q4 zero = {{0.f, 0.f, 0.f, 0.f}};
    const int64_t r0 = (int64_t)blockIdx.x * R;
    u32x4 rx[R], ry[R];
    int64_t row[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        row[i] = r0 + i < p.rows ? r0 + i : p.rows - 1;                  // (behind the last row: that row once more, not stored)
        rx[i] = ry[i] = (u32x4){0u, 0u, 0u, 0u};
    }
    if (on) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            rx[i] = rn_raw<VEC, XT, NT>(rn_row<XT>((const char*)p.x, p.x_dt, row[i] * p.cols), p.x_dt, c, p.cols);
            ry[i] = rn_raw<VEC, YT, NT>(rn_row<YT>((const char*)p.y, p.y_dt, row[i] * p.cols), p.y_dt, c, p.cols);
        }
    }
    rn_clear(red);
    int turn = 0;
    Q4 g1 = zero, b1 = zero, g2 = zero, b2 = zero, gate[R];
    if (p.g1) { g1 = rn_param<VEC>(p.g1, 0, c, p.cols); if (p.b1) b1 = rn_param<VEC>(p.b1, 0, c, p.cols); }
    if (p.g2) { g2 = rn_param<VEC>(p.g2, 0, c, p.cols); if (p.b2) b2 = rn_param<VEC>(p.b2, 0, c, p.cols); }
    if (p.gate_kind == HH_GATE_GROUP) {
#pragma unroll
        for (int i = 0; i < R; ++i) gate[i] = rn_gate<VEC>(p, row[i] / p.each, c);
    } else {
        gate[0] = rn_gate<VEC>(p, 0, c);
#pragma unroll
        for (int i = 1; i < R; ++i) gate[i] = gate[0];
    }
    Q4 x[R], y[R];
    float mean[R], rstd[R], eps[R];
#pragma unroll
    for (int i = 0; i < R; ++i) { x[i] = rn_cvt<VEC, XT>(rx[i], p.x_dt, behind); y[i] = rn_cvt<VEC, YT>(ry[i], p.y_dt, behind); }
    if (p.g1) {
#pragma unroll
        for (int i = 0; i < R; ++i) eps[i] = p.eps1;
        rn_stats<VEC, true, R>(y, c, p.cols, inv, p.rms, eps, red, turn, waves, mean, rstd);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) y[i].v[j] = (y[i].v[j] - mean[i]) * rstd[i] * g1.v[j] + b1.v[j];
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i].v[j] = x[i].v[j] * p.res_scale + gate[i].v[j] * y[i].v[j];
        if (r0 + i < p.rows && on) rn_store<VEC, NT, XT>(x[i], rn_row<XT>((char*)p.x_new, p.x_dt, row[i] * p.cols), p.x_dt, c, p.cols);
    }
    if (p.g2) {
#pragma unroll
        for (int i = 0; i < R; ++i) eps[i] = p.eps2;
        rn_stats<VEC, false, R>(x, c, p.cols, inv, p.rms, eps, red, turn, waves, mean, rstd);
#pragma unroll
        for (int i = 0; i < R; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i].v[j] = (x[i].v[j] - mean[i]) * rstd[i] * g2.v[j] + b2.v[j];
            if (r0 + i < p.rows && on) rn_store<VEC, NT, HT>(x[i], rn_row<HT>((char*)p.h, p.h_dt, row[i] * p.cols), p.h_dt, c, p.cols);
        }
    }
}

// (four rows at a time take 192 registers: for up to 1024 channels, whose workgroups have no more than four waves)
template <int R, bool POST, bool PRE, bool VEC, bool NT, int XT, int YT, int HT>
__global__ __launch_bounds__(R == 4 ? 256 : 1024) void resnorm_bwd_kernel(RnParams p) {
    __shared__ RnRed red;
    const int waves = blockDim.x >> 6, c = threadIdx.x * 4, behind = rn_behind(c, p.cols);
    const bool on = c < p.cols;
    const float inv = 1.f / (float)p.cols;
    const Q4 zero = {{0.f, 0.f, 0.f, 0.f}};
    const u32x4 none = {0u, 0u, 0u, 0u};
    rn_clear(red);
    int turn = 0;
    Q4 g2 = zero, ag1 = zero, ab1 = zero, ag2 = zero, ab2 = zero;
    if (PRE) g2 = rn_param<VEC>(p.g2, 0, c, p.cols);
    const int64_t u0 = blockIdx.x * p.per_block, u1 = u0 + p.per_block < p.units ? u0 + p.per_block : p.units;
    for (int64_t u = u0; u < u1; ++u) {
        const int64_t group = u / p.chunks, first = group * p.each + (u % p.chunks) * R, last = (group + 1) * p.each;
        const Q4 gate = rn_gate<VEC>(p, group, c);
        Q4 w = gate, s0 = zero, s1 = zero;                               // w: g o gamma of post
        if (POST) {
            w = rn_param<VEC>(p.g1, 0, c, p.cols);
#pragma unroll
            for (int j = 0; j < 4; ++j) w.v[j] *= gate.v[j];
        }
        for (int64_t r = first; r < last; r += p.chunks * R) {
            u32x4 rx[R], rh[R], rd[R], ry[R];
#pragma unroll
            for (int i = 0; i < R; ++i) rx[i] = rh[i] = rd[i] = ry[i] = none;
            if (on) {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    // behind the group's last row: that row once more, with gradients of zero, and not stored
                    const int64_t off = (r + i < last ? r + i : last - 1) * p.cols;
                    if (PRE) rx[i] = rn_raw<VEC, XT, NT>(rn_row<XT>((const char*)p.x_new, p.x_dt, off), p.x_dt, c, p.cols);
                    ry[i] = rn_raw<VEC, YT, NT>(rn_row<YT>((const char*)p.y, p.y_dt, off), p.y_dt, c, p.cols);
                    if (i == 0 || r + i < last) {
                        if (PRE) rh[i] = rn_raw<VEC, HT, NT>(rn_row<HT>((const char*)p.dh, p.h_dt, off), p.h_dt, c, p.cols);
                        if (p.dx_new) rd[i] = rn_raw<VEC, XT, NT>(rn_row<XT>((const char*)p.dx_new, p.x_dt, off), p.x_dt, c, p.cols);
                    }
                }
            }
            float mean[2 * R], rstd[2 * R], s[2 * R];
            Q4 y[R], d[R];
            if constexpr (PRE) {
                Q4 x[R];
                if constexpr (POST) {                                    // both norms' statistics in the same two exchanges
                    Q4 xy[2 * R];
                    float eps[2 * R];
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        xy[i] = rn_cvt<VEC, XT>(rx[i], p.x_dt, behind); xy[R + i] = rn_cvt<VEC, YT>(ry[i], p.y_dt, behind);
                        eps[i] = p.eps2; eps[R + i] = p.eps1;
                    }
                    rn_stats<VEC, true, 2 * R>(xy, c, p.cols, inv, p.rms, eps, red, turn, waves, mean, rstd);
#pragma unroll
                    for (int i = 0; i < R; ++i) { x[i] = xy[i]; y[i] = xy[R + i]; }
                } else {
                    float eps[R], m[R], q[R];
#pragma unroll
                    for (int i = 0; i < R; ++i) { x[i] = rn_cvt<VEC, XT>(rx[i], p.x_dt, behind); y[i] = rn_cvt<VEC, YT>(ry[i], p.y_dt, behind); eps[i] = p.eps2; }
                    rn_stats<VEC, true, R>(x, c, p.cols, inv, p.rms, eps, red, turn, waves, m, q);
#pragma unroll
                    for (int i = 0; i < R; ++i) { mean[i] = m[i]; rstd[i] = q[i]; }
                }
                Q4 k[R];
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    k[i] = rn_cvt<VEC, HT>(rh[i], p.h_dt, behind);
                    d[i] = rn_cvt<VEC, XT>(rd[i], p.x_dt, behind);
                    s[i] = s[R + i] = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float xh = (x[i].v[j] - mean[i]) * rstd[i];
                        ag2.v[j] += k[i].v[j] * xh;
                        ab2.v[j] += k[i].v[j];
                        k[i].v[j] *= g2.v[j];                            // (channels behind the row's end: dh and gamma are zero there)
                        s[i] += k[i].v[j];
                        s[R + i] += k[i].v[j] * xh;
                        x[i].v[j] = xh;
                    }
                }
                block_sums<2 * R>(s, red, turn, waves);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float a = p.rms ? 0.f : s[i] * inv, b = s[R + i] * inv;
#pragma unroll
                    for (int j = 0; j < 4; ++j) d[i].v[j] += rstd[i] * (k[i].v[j] - a - x[i].v[j] * b);
                }
            } else {
#pragma unroll
                for (int i = 0; i < R; ++i) { y[i] = rn_cvt<VEC, YT>(ry[i], p.y_dt, behind); d[i] = rn_cvt<VEC, XT>(rd[i], p.x_dt, behind); }
                if constexpr (POST) {
                    float eps[R], m[R], q[R];
#pragma unroll
                    for (int i = 0; i < R; ++i) eps[i] = p.eps1;
                    rn_stats<VEC, true, R>(y, c, p.cols, inv, p.rms, eps, red, turn, waves, m, q);
#pragma unroll
                    for (int i = 0; i < R; ++i) { mean[R + i] = m[i]; rstd[R + i] = q[i]; }
                }
            }
            // (a row behind the group's last has d = 0 - rstd * (0 - 0 - xh * 0) = 0: its gradients are zero, so it adds nothing below either)
            if constexpr (POST) {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    s[i] = s[R + i] = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float xh = (y[i].v[j] - mean[R + i]) * rstd[R + i];
                        s0.v[j] += d[i].v[j];
                        s1.v[j] += d[i].v[j] * xh;
                        const float k = d[i].v[j] * w.v[j];              // (channels behind the row's end: w is zero there)
                        s[i] += k;
                        s[R + i] += k * xh;
                        y[i].v[j] = xh;
                    }
                }
                block_sums<2 * R>(s, red, turn, waves);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float a = p.rms ? 0.f : s[i] * inv, b = s[R + i] * inv;
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[i].v[j] = rstd[R + i] * (d[i].v[j] * w.v[j] - a - y[i].v[j] * b);
                }
            } else {
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s1.v[j] += d[i].v[j] * y[i].v[j];
                        y[i].v[j] = d[i].v[j] * w.v[j];
                    }
            }
            if (on) {
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (i == 0 || r + i < last) {
                        const int64_t off = (r + i) * p.cols;
                        rn_store<VEC, NT, YT>(y[i], rn_row<YT>((char*)p.dy, p.y_dt, off), p.y_dt, c, p.cols);
#pragma unroll
                        for (int j = 0; j < 4; ++j) d[i].v[j] *= p.res_scale;
                        rn_store<VEC, NT, XT>(d[i], rn_row<XT>((char*)p.dx, p.x_dt, off), p.x_dt, c, p.cols);
                    }
            }
        }
        Q4 t = s1;                                                       // the unit's share of the gate's gradient: sum d o p
        if constexpr (POST) {
            const Q4 g1 = rn_param<VEC>(p.g1, 0, c, p.cols);
            const Q4 b1 = p.b1 ? rn_param<VEC>(p.b1, 0, c, p.cols) : zero;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                ag1.v[j] += gate.v[j] * s1.v[j];
                ab1.v[j] += gate.v[j] * s0.v[j];
                t.v[j] = g1.v[j] * s1.v[j] + b1.v[j] * s0.v[j];
            }
        }
        if (p.gate_kind == HH_GATE_SCALAR) {
            float sum[1] = {rn_sum4<false>(t, c, p.cols)};
            block_sums<1>(sum, red, turn, waves);
            if (threadIdx.x == 0) p.gate_part[u] = sum[0];
        } else if (p.gate_kind != HH_GATE_NONE) {
            rn_put<VEC>(t, p.gate_part + u * p.cols, c, p.cols);
        }
    }
    const int64_t plane = (int64_t)gridDim.x * p.cols;
    float* out = p.part + blockIdx.x * (int64_t)p.cols;
    if constexpr (POST) {
        rn_put<VEC>(ag1, out, c, p.cols);
        if (p.b1) rn_put<VEC>(ab1, out + plane, c, p.cols);             // (a norm without beta: no plane of its gradient)
    }
    if constexpr (PRE) {
        rn_put<VEC>(ag2, out + 2 * plane, c, p.cols);
        if (p.b2) rn_put<VEC>(ab2, out + 3 * plane, c, p.cols);
    }
}

// The second launch: column sums of the partial rows.  Three kinds of workgroups, told apart by blockIdx.x:
//   [0, planes * cols16): a plane of the norms' gradients (or, for up to RN_WIDE_GROUPS gate groups, such a group's rows), 16 channels; 64 lanes share a channel's
//                         rows, eight loads in flight each
//   then the gate groups, where there are more of them and so few rows in each that a thread takes a channel of a group by itself
//   then one workgroup for a scalar gate's sum.
#define RN_WIDE_GROUPS 32
struct RnReduce {
    const float* part[4]; float* out[4];   // the planes that are wanted
    const float* gate_part; const float* gate; float* dgate;
    int64_t blocks, chunks, units, groups;
    int planes, cols, cols16, gate_kind, gate_tanh, wide_groups;
    int64_t first_narrow, first_scalar;
};
__device__ __forceinline__ float rn_untanh(const RnReduce& p, int64_t at, float s) {
    if (p.gate_tanh) { const float th = tanhf(p.gate[at]); s *= 1.f - th * th; }
    return s;
}
__global__ __launch_bounds__(1024) void resnorm_reduce_kernel(RnReduce p) {
    __shared__ float buf[16][16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (blockIdx.x < p.first_narrow) {
        const int which = blockIdx.x / p.cols16, c = (blockIdx.x % p.cols16) * 16 + (lane & 15);
        const bool is_gate = which >= p.planes;
        const int64_t group = which - p.planes, n = is_gate ? p.chunks : p.blocks;
        const float* src = (is_gate ? p.gate_part + group * p.chunks * p.cols : p.part[which]) + c;
        float s = 0.f;
        if (c < p.cols)
            for (int64_t r = wave * 4 + (lane >> 4); r < n; r += 64 * 8) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = r + 64 * i < n ? src[(r + 64 * i) * p.cols] : 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += v[i];
            }
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (lane < 16) buf[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && lane < 16 && c < p.cols) {
            s = 0.f;
#pragma unroll
            for (int w = 0; w < 16; ++w) s += buf[w][lane];
            if (is_gate) p.dgate[group * p.cols + c] = rn_untanh(p, group * p.cols + c, s);
            else p.out[which][c] = s;
        }
    } else if (blockIdx.x < p.first_scalar) {
        const int64_t i = ((int64_t)blockIdx.x - p.first_narrow) * 1024 + threadIdx.x;
        if (i >= p.groups * p.cols) return;
        const int64_t group = i / p.cols;
        const float* src = p.gate_part + group * p.chunks * p.cols + i % p.cols;
        float s = 0.f;
        for (int64_t r = 0; r < p.chunks; r += 8) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = r + k < p.chunks ? src[(r + k) * p.cols] : 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) s += v[k];
        }
        p.dgate[i] = rn_untanh(p, i, s);
    } else {
        float s = 0.f;
        for (int64_t i = threadIdx.x; i < p.units; i += 1024) s += p.gate_part[i];
        s = wave_sum(s);
        if (lane == 0) buf[wave][0] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            s = 0.f;
            for (int w = 0; w < 16; ++w) s += buf[w][0];
            p.dgate[0] = rn_untanh(p, 0, s);
        }
    }
}

// ---- entry points ------------------------------------------------------------------------------------------------------------------------
// rows from which the forward pass takes four at a time (4097 x 1024: 10.8 us, one at a time 11.7; 32 776 x 1024: 66 and 75) and below which it takes one, where a
// call is all latency (416 x 512: 3.6 us, four at a time 4.3)
#define RN_FWD_MANY 4096
static int rn_waves(int cols) { return (cols + 255) / 256; }

struct RnPlan { int64_t chunks, units, per_block, blocks; };
// Workgroups that are on the chip at once (two rows at a time: 16 waves to a CU, four rows: 8), which take whole units of one gate group's rows.  A unit leaves four
// partial rows, so it has 8 rows (12 320 x 768: 4 rows 35.1 us, 8 rows 35.2, 16 rows 37.0; the caller's other operands matter as much: 33.0 and 34.6 us for 8 and 16) --
// fewer where that gives less than a workgroup to a CU, down to the two that are worked on at once (416 x 512: 8 rows 12.6 us, 2 rows 8.6; 1024 x 1024: 2 rows 19.0,
// 4 rows 14.0, 8 rows 15.5).
static RnPlan rn_plan(int64_t rows, int cols, int64_t groups, int at_once) {
    RnPlan q;
    const int64_t blocks = 256 * ((at_once == 4 ? 8 : 16) / rn_waves(cols));
    const int64_t each = rows / groups, few = (255 + groups) / groups, pairs = (each + 1) / 2;
    const int64_t most = (each + 7) / 8, least = pairs < few ? pairs : few;
    q.chunks = (blocks + groups - 1) / groups;
    if (q.chunks > most) q.chunks = most > least ? most : least;
    q.units = q.chunks * groups;
    q.per_block = (q.units + blocks - 1) / blocks;
    q.blocks = (q.units + q.per_block - 1) / q.per_block;
    return q;
}

static int rn_check(const hh_residual_norm* d, bool bwd, const char* who) {
    HH_REQUIRE(d != nullptr, HH_ERR_SHAPE, "%s: NULL description", who);
    HH_REQUIRE(d->rows >= 0 && d->rows < (1ll << 40) && d->cols > 0 && d->cols <= 4096, HH_ERR_SHAPE, "%s: cols=%d must be in [1, 4096], rows=%lld below 2^40", who, d->cols, (long long)d->rows);
    HH_REQUIRE(d->gate_kind >= HH_GATE_NONE && d->gate_kind <= HH_GATE_GROUP, HH_ERR_UNSUPPORTED, "%s: unknown gate kind %d", who, d->gate_kind);
    HH_REQUIRE(d->groups >= 1 && d->groups <= 65000 && d->rows % d->groups == 0 && (d->groups == 1 || d->gate_kind == HH_GATE_GROUP), HH_ERR_SHAPE,
               "%s: %lld rows do not split into %lld gate groups (1 without a gate for each group, 65000 at most)", who, (long long)d->rows, (long long)d->groups);
    HH_REQUIRE((d->x_dtype == HH_F32 || d->x_dtype == HH_BF16) && (d->y_dtype == HH_F32 || d->y_dtype == HH_BF16) && (d->h_dtype == HH_F32 || d->h_dtype == HH_BF16), HH_ERR_DTYPE,
               "%s: bad dtype", who);
    // (the parameters are read without rows too: the backward pass of none writes their gradients, a tanh gate's from its values)
    HH_REQUIRE((d->gate_kind == HH_GATE_NONE) == (d->gate == nullptr), HH_ERR_ALIGN, "%s: gate kind and pointer do not agree", who);
    HH_REQUIRE(d->post_gamma != nullptr || d->post_beta == nullptr, HH_ERR_ALIGN, "%s: post_beta without post_gamma", who);
    HH_REQUIRE(d->pre_gamma != nullptr || d->pre_beta == nullptr, HH_ERR_ALIGN, "%s: pre_beta without pre_gamma", who);
    if (d->rows == 0) return HH_OK;
    HH_REQUIRE(d->y != nullptr && d->x_new != nullptr && (bwd ? (d->dx != nullptr && d->dy != nullptr) : d->x != nullptr), HH_ERR_ALIGN, "%s: NULL pointer", who);
    if (bwd) HH_REQUIRE((d->dh != nullptr) == (d->pre_gamma != nullptr), HH_ERR_ALIGN, "%s: dh comes with pre_gamma", who);
    else HH_REQUIRE((d->h != nullptr) == (d->pre_gamma != nullptr), HH_ERR_ALIGN, "%s: h comes with pre_gamma", who);
    return HH_OK;
}

static RnParams rn_params(const hh_residual_norm* d, bool* vec) {
    RnParams p;
    p.x = d->x; p.y = d->y; p.x_new = d->x_new; p.h = d->h; p.dx_new = d->dx_new; p.dh = d->dh; p.dx = d->dx; p.dy = d->dy;
    p.gate = d->gate; p.g1 = d->post_gamma; p.b1 = d->post_beta; p.g2 = d->pre_gamma; p.b2 = d->pre_beta;
    p.part = p.gate_part = nullptr;
    p.rows = d->rows; p.each = d->rows / d->groups; p.chunks = p.units = p.per_block = 0;
    p.cols = d->cols; p.gate_kind = d->gate_kind; p.gate_tanh = d->gate_tanh; p.rms = d->rms;
    p.x_dt = d->x_dtype; p.y_dt = d->y_dtype; p.h_dt = d->h_dtype;
    p.eps1 = d->post_eps; p.eps2 = d->pre_eps; p.res_scale = d->res_scale;
    *vec = d->cols % 4 == 0 && HH_ALIGNED16(p.x) && HH_ALIGNED16(p.y) && HH_ALIGNED16(p.x_new) && HH_ALIGNED16(p.h) && HH_ALIGNED16(p.dx_new) && HH_ALIGNED16(p.dh) && HH_ALIGNED16(p.dx) &&
           HH_ALIGNED16(p.dy) && (d->gate_kind == HH_GATE_SCALAR || HH_ALIGNED16(p.gate)) && HH_ALIGNED16(p.g1) && HH_ALIGNED16(p.b1) && HH_ALIGNED16(p.g2) && HH_ALIGNED16(p.b2);
    return p;
}
static int64_t rn_size(int dtype) { return dtype == HH_F32 ? 4 : 2; }

extern "C" int hh_residual_norm_fwd(const hh_residual_norm* d, hh_stream_t stream) {
    const int rc = rn_check(d, false, "hh_residual_norm_fwd");
    if (rc != HH_OK || d->rows == 0) return rc;
    hipStream_t s = (hipStream_t)stream;
    bool vec;
    const RnParams p = rn_params(d, &vec);
    const bool nt = d->rows * d->cols * (rn_size(p.x_dt) + (p.h ? rn_size(p.h_dt) : 0)) > HH_STREAM_BYTES;
    const int threads = rn_waves(p.cols) * 64;
    HH_REQUIRE(hh_grid_fits(d->rows < RN_FWD_MANY ? d->rows : (d->rows + 3) / 4, threads), HH_ERR_SHAPE, "hh_residual_norm_fwd: too many rows for a launch (rows=%lld cols=%d)", (long long)d->rows, p.cols);
#define RF(R, V, N, X, Y, H) hipLaunchKernelGGL((resnorm_fwd_kernel<R, V, N, X, Y, H>), dim3((unsigned)((d->rows + R - 1) / R)), dim3(threads), 0, s, p)
#define RFN(X, Y, H) do { if (d->rows < RN_FWD_MANY) RF(1, true, false, X, Y, H); else if (nt) RF(4, true, true, X, Y, H); else RF(4, true, false, X, Y, H); } while (0)
#define RFH(X, Y) do { if (p.h_dt == HH_F32) RFN(X, Y, HH_F32); else RFN(X, Y, HH_BF16); } while (0)
    if (!vec) { if (d->rows < RN_FWD_MANY) RF(1, false, false, RN_ANY, RN_ANY, RN_ANY); else if (nt) RF(4, false, true, RN_ANY, RN_ANY, RN_ANY); else RF(4, false, false, RN_ANY, RN_ANY, RN_ANY); }
    else if (p.x_dt == HH_F32) { if (p.y_dt == HH_F32) RFH(HH_F32, HH_F32); else RFH(HH_F32, HH_BF16); }
    else { if (p.y_dt == HH_F32) RFH(HH_BF16, HH_F32); else RFH(HH_BF16, HH_BF16); }
#undef RFH
#undef RFN
#undef RF
    return hh_check_launch("hh_residual_norm_fwd");
}

extern "C" int64_t hh_workspace_bytes_residual_norm_bwd(int64_t rows, int cols, int64_t groups) {
    if (rows < 0 || cols <= 0 || cols > 4096 || groups < 1 || groups > 65000 || rows % groups) return -1;
    if (rows == 0) return 0;
    const RnPlan q = rn_plan(rows, cols, groups, 2), q4 = cols <= 1024 ? rn_plan(rows, cols, groups, 4) : q;
    const int64_t lines = 4 * q.blocks + q.units, lines4 = 4 * q4.blocks + q4.units;
    return (lines > lines4 ? lines : lines4) * cols * 4;
}

extern "C" int hh_residual_norm_bwd(const hh_residual_norm* d, hh_stream_t stream) {
    const int rc = rn_check(d, true, "hh_residual_norm_bwd");
    if (rc != HH_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    bool vec;
    RnParams p = rn_params(d, &vec);
    HH_REQUIRE((p.gate_kind == HH_GATE_NONE) == (d->dgate == nullptr) && (p.g1 != nullptr) == (d->dpost_gamma != nullptr) && (p.g2 != nullptr) == (d->dpre_gamma != nullptr) &&
                   (p.b1 != nullptr || d->dpost_beta == nullptr) && (p.b2 != nullptr || d->dpre_beta == nullptr),
               HH_ERR_ALIGN, "hh_residual_norm_bwd: a gradient's pointer comes with its parameter's");
    RnPlan q = {0, 0, 0, 0};                                     // (no rows: every sum is over nothing, and the second launch writes zeros)
    if (d->rows > 0) {
        // two rows at a time, and four for the largest calls of up to 1024 channels: their requests are larger, but their workgroups fill the chip only where they have
        // one, two or four waves, and a few hundred MB of gradients have to be written before that pays (1024 channels: 35 807 rows 138 us, four 141; 65 104 rows 238
        // and 242; 130 208 rows 497 and 473.  768 channels: 173 611 rows 491 and 533)
        const int64_t bytes = d->rows * p.cols * (rn_size(p.x_dt) + rn_size(p.y_dt));
        const bool nt = bytes > HH_STREAM_BYTES;
        const int waves = rn_waves(p.cols), threads = waves * 64, at_once = vec && bytes > (600ll << 20) && (waves == 1 || waves == 2 || waves == 4) ? 4 : 2;
        q = rn_plan(d->rows, p.cols, d->groups, at_once);
        HH_REQUIRE(d->workspace != nullptr && HH_ALIGNED16(d->workspace), HH_ERR_ALIGN, "hh_residual_norm_bwd: a 16-byte aligned workspace is needed");
        p.part = (float*)d->workspace;
        p.gate_part = p.part + 4 * q.blocks * p.cols;
        p.chunks = q.chunks; p.units = q.units; p.per_block = q.per_block;
#define RB(R, PO, PR, V, N, X, Y, H) hipLaunchKernelGGL((resnorm_bwd_kernel<R, PO, PR, V, N, X, Y, H>), dim3((unsigned)q.blocks), dim3(threads), 0, s, p)
#define RBN(PO, PR, X, Y, H) do { if (at_once == 4) RB(4, PO, PR, true, true, X, Y, H); else if (nt) RB(2, PO, PR, true, true, X, Y, H); else RB(2, PO, PR, true, false, X, Y, H); } while (0)
#define RBY(PO, PR, X, H) do { if (p.y_dt == HH_F32) RBN(PO, PR, X, HH_F32, H); else RBN(PO, PR, X, HH_BF16, H); } while (0)
#define RBX(PO, PR, H) do { if (!vec) { if (nt) RB(2, PO, PR, false, true, RN_ANY, RN_ANY, RN_ANY); else RB(2, PO, PR, false, false, RN_ANY, RN_ANY, RN_ANY); } else if (p.x_dt == HH_F32) RBY(PO, PR, HH_F32, H); else RBY(PO, PR, HH_BF16, H); } while (0)
        if (p.g1 && p.g2) { if (p.h_dt == HH_F32) RBX(true, true, HH_F32); else RBX(true, true, HH_BF16); }
        else if (p.g2) { if (p.h_dt == HH_F32) RBX(false, true, HH_F32); else RBX(false, true, HH_BF16); }
        else if (p.g1) RBX(true, false, HH_F32);
        else RBX(false, false, HH_F32);
#undef RBX
#undef RBY
#undef RBN
#undef RB
    }
    RnReduce r;
    r.planes = 0;
    float* outs[4] = {d->dpost_gamma, d->dpost_beta, d->dpre_gamma, d->dpre_beta};
    for (int i = 0; i < 4; ++i)
        if (outs[i]) {
            r.part[r.planes] = p.part + (int64_t)i * q.blocks * p.cols;
            r.out[r.planes++] = outs[i];
        }
    r.gate_part = p.gate_part; r.gate = p.gate; r.dgate = d->dgate;
    r.blocks = q.blocks; r.chunks = q.chunks; r.units = q.units; r.groups = d->groups;
    r.cols = p.cols; r.cols16 = (p.cols + 15) / 16; r.gate_kind = p.gate_kind; r.gate_tanh = p.gate_tanh;
    const bool rowed = p.gate_kind == HH_GATE_CHANNEL || p.gate_kind == HH_GATE_GROUP;
    r.wide_groups = rowed && d->groups <= RN_WIDE_GROUPS ? (int)d->groups : 0;
    r.first_narrow = (int64_t)(r.planes + r.wide_groups) * r.cols16;
    r.first_scalar = r.first_narrow + (rowed && !r.wide_groups ? (d->groups * p.cols + 1023) / 1024 : 0);
    const int64_t grid = r.first_scalar + (p.gate_kind == HH_GATE_SCALAR);
    if (grid) hipLaunchKernelGGL(resnorm_reduce_kernel, dim3((unsigned)grid), dim3(1024), 0, s, r);
    return hh_check_launch("hh_residual_norm_bwd");
}
