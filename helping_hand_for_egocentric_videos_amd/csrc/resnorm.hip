// The end of a residual block in one pass over its rows, and its gradients:
//     p = post(y)  (a norm, or y itself),   x_new = res_scale * x + g o p,   h = pre(x_new)  (the next block's norm, or nothing)
// where a norm is gamma o (v - mean) * rstd + beta (LayerNorm) or gamma o v * rrms (+ beta), and the gate g is 1, a scalar, a row over the
// channels, or such a row for each group of consecutive rows, as it is or through tanh (the tanh gate of model/LaviLa.py:305-390 is the scalar one).
// Statistics are two-pass and in fp32, from the fp32 x_new before it is rounded to its storage type.
//
// Backward, from x_new, y and the gradients dx_new, dh (statistics are taken again: both rows are in registers anyway, and nothing has to be kept):
//     d = dx_new + pre'(dh),   dx = res_scale * d,   dgate = sum d o p (* 1 - tanh^2),   dy = post'(g o d),
//     n'(dn) = rstd * (k - mean(k) - xh * mean(k o xh)) with k = dn o gamma and xh the normed row   (no mean(k) term for root-mean-square norms).
// Gradients of gamma, beta and the gate are column sums: every workgroup sums its rows in registers and leaves one row of partial sums, which a
// second launch adds in workgroup order (no atomics: equal inputs give equal bits).
#include "common.h"

// cols <= WPR * NV * 256: WPR waves share a row, each lane holds NV pieces of 4 consecutive channels
template <int NV>
struct Row { float v[NV][4]; };

struct RnParams {
    const void* x; const void* y; void* x_new; void* h;
    const void* dx_new; const void* dh; void* dx; void* dy;
    const float* gate; const float* g1; const float* b1; const float* g2; const float* b2;
    float* part;                       // [4][blocks][cols]: dgamma / dbeta of post, of pre;  behind them [units][cols] (or [units]) of the gate
    float* gate_part;
    int64_t rows, each;                // rows of one gate group (all of them without groups)
    int64_t chunk, chunks;             // rows of a unit, units of a group
    int64_t units, per_block;          // units in all, and of one workgroup
    int cols, gate_kind, gate_tanh, rms, vec;
    int x_dt, y_dt, h_dt;
    float eps1, eps2, res_scale;
};

template <int NV, int WPR>
__device__ __forceinline__ void rn_load(Row<NV>& r, const void* base, int dt, int64_t off, int cols, int vec, int t) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WPR + t) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) r.v[i][j] = 0.f;
        if (c < cols) {
            if (vec) {
                if (dt == HH_F32) {
                    const f32x4 q = *(const f32x4*)((const float*)base + off + c);
#pragma unroll
                    for (int j = 0; j < 4; ++j) r.v[i][j] = q[j];
                } else {
                    const u32x2 q = *(const u32x2*)((const bf16_t*)base + off + c);
                    r.v[i][0] = bf16_lo_to_f32(q[0]); r.v[i][1] = bf16_hi_to_f32(q[0]);
                    r.v[i][2] = bf16_lo_to_f32(q[1]); r.v[i][3] = bf16_hi_to_f32(q[1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < cols) r.v[i][j] = dt == HH_F32 ? ((const float*)base)[off + c + j] : (float)((const bf16_t*)base)[off + c + j];
            }
        }
    }
}
template <int NV, int WPR>
__device__ __forceinline__ void rn_store(const Row<NV>& r, void* base, int dt, int64_t off, int cols, int vec, int t) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * WPR + t) * 4;
        if (c < cols) {
            if (vec) {
                if (dt == HH_F32) {
                    const f32x4 q = {r.v[i][0], r.v[i][1], r.v[i][2], r.v[i][3]};
                    *(f32x4*)((float*)base + off + c) = q;
                } else {
                    const u32x2 q = {pack_bf16(r.v[i][0], r.v[i][1]), pack_bf16(r.v[i][2], r.v[i][3])};
                    *(u32x2*)((bf16_t*)base + off + c) = q;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < cols) {
                        if (dt == HH_F32) ((float*)base)[off + c + j] = r.v[i][j];
                        else ((bf16_t*)base)[off + c + j] = (bf16_t)r.v[i][j];
                    }
            }
        }
    }
}

// sums of N values over the WPR waves of a row; `red` holds [4 waves][N], and the two barriers keep its uses apart
template <int N, int WPR>
__device__ __forceinline__ void row_sums(float (&s)[N], float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) s[k] += __shfl_xor(s[k], o, 64);
    if constexpr (WPR > 1) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) red[wave * N + k] = s[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            s[k] = 0.f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) s[k] += red[w * N + k];
        }
        __syncthreads();
    }
}

template <int NV, int WPR>
__device__ __forceinline__ bool rn_in(int i, int j, int t, int cols) { return (i * 64 * WPR + t) * 4 + j < cols; }

// means and reciprocal standard deviations of two rows at once (one reduction tree for both)
template <int NV, int WPR>
__device__ __forceinline__ void rn_stats2(const Row<NV>& a, const Row<NV>& b, int cols, int rms, float eps_a, float eps_b, int t, float* red, float (&mean)[2], float (&rstd)[2]) {
    const float inv = 1.f / (float)cols;
    mean[0] = mean[1] = 0.f;
    if (!rms) {
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) { s[0] += a.v[i][j]; s[1] += b.v[i][j]; }
        row_sums<2, WPR>(s, red);
        mean[0] = s[0] * inv; mean[1] = s[1] * inv;
    }
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (rn_in<NV, WPR>(i, j, t, cols)) {
                const float da = a.v[i][j] - mean[0], db = b.v[i][j] - mean[1];
                q[0] += da * da; q[1] += db * db;
            }
    row_sums<2, WPR>(q, red);
    rstd[0] = 1.f / sqrtf(q[0] * inv + eps_a);
    rstd[1] = 1.f / sqrtf(q[1] * inv + eps_b);
}
template <int NV, int WPR>
__device__ __forceinline__ void rn_stats(const Row<NV>& a, int cols, int rms, float eps, int t, float* red, float& mean, float& rstd) {
    const float inv = 1.f / (float)cols;
    mean = 0.f;
    if (!rms) {
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[0] += a.v[i][j];
        row_sums<1, WPR>(s, red);
        mean = s[0] * inv;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (rn_in<NV, WPR>(i, j, t, cols)) { const float d = a.v[i][j] - mean; q[0] += d * d; }
    row_sums<1, WPR>(q, red);
    rstd = 1.f / sqrtf(q[0] * inv + eps);
}

template <int NV, int WPR>
__device__ __forceinline__ void rn_gate(Row<NV>& g, const RnParams& p, int64_t group, int t) {
    if (p.gate_kind == HH_GATE_NONE) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) g.v[i][j] = 1.f;
        return;
    }
    if (p.gate_kind == HH_GATE_SCALAR) {
        const float a = p.gate_tanh ? tanhf(p.gate[0]) : p.gate[0];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) g.v[i][j] = a;
        return;
    }
    rn_load<NV, WPR>(g, p.gate, HH_F32, p.gate_kind == HH_GATE_GROUP ? group * p.cols : 0, p.cols, p.vec, t);
    if (p.gate_tanh)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) g.v[i][j] = tanhf(g.v[i][j]);
}

template <int NV, int WPR, bool POST, bool PRE>
__global__ __launch_bounds__(256) void resnorm_fwd_kernel(RnParams p) {
    __shared__ float red[8];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int t = WPR == 1 ? lane : (int)threadIdx.x;
    const int64_t row = WPR == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x;
    if (row >= p.rows) return;                       // (a whole wave, and with WPR = 4 no block at all: its barriers are met by every wave)
    const int64_t off = row * p.cols;
    Row<NV> x, y, k;
    rn_load<NV, WPR>(x, p.x, p.x_dt, off, p.cols, p.vec, t);
    rn_load<NV, WPR>(y, p.y, p.y_dt, off, p.cols, p.vec, t);
    if constexpr (POST) {
        float mean, rstd;
        rn_stats<NV, WPR>(y, p.cols, p.rms, p.eps1, t, red, mean, rstd);
        rn_load<NV, WPR>(k, p.g1, HH_F32, 0, p.cols, p.vec, t);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) y.v[i][j] = (y.v[i][j] - mean) * rstd * k.v[i][j];
        if (p.b1) {
            rn_load<NV, WPR>(k, p.b1, HH_F32, 0, p.cols, p.vec, t);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) y.v[i][j] += k.v[i][j];
        }
    }
    rn_gate<NV, WPR>(k, p, row / p.each, t);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) x.v[i][j] = x.v[i][j] * p.res_scale + k.v[i][j] * y.v[i][j];
    rn_store<NV, WPR>(x, p.x_new, p.x_dt, off, p.cols, p.vec, t);
    if constexpr (PRE) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (!rn_in<NV, WPR>(i, j, t, p.cols)) x.v[i][j] = 0.f;          // (channels behind the row's end: 0 * inf above would be NaN)
        float mean, rstd;
        rn_stats<NV, WPR>(x, p.cols, p.rms, p.eps2, t, red, mean, rstd);
        rn_load<NV, WPR>(k, p.g2, HH_F32, 0, p.cols, p.vec, t);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) x.v[i][j] = (x.v[i][j] - mean) * rstd * k.v[i][j];
        if (p.b2) {
            rn_load<NV, WPR>(k, p.b2, HH_F32, 0, p.cols, p.vec, t);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) x.v[i][j] += k.v[i][j];
        }
        rn_store<NV, WPR>(x, p.h, p.h_dt, off, p.cols, p.vec, t);
    }
}

// column sums of the four waves (WPR = 1: each saw rows of its own) or of the row's four waves (WPR = 4: each owns its channels) -> one fp32 row
template <int NV, int WPR>
__device__ __forceinline__ void rn_put_cols(const Row<NV>& a, float* out, int cols, int t, float* buf) {
    const int wave = threadIdx.x >> 6;
    if constexpr (WPR == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) buf[wave * NV * 256 + (i * 64 + t) * 4 + j] = a.v[i][j];
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += 256) out[c] = (buf[c] + buf[NV * 256 + c]) + (buf[2 * NV * 256 + c] + buf[3 * NV * 256 + c]);
        __syncthreads();
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (rn_in<NV, WPR>(i, j, t, cols)) out[(i * 64 * WPR + t) * 4 + j] = a.v[i][j];
    }
}

template <int NV, int WPR, bool POST, bool PRE>
__global__ __launch_bounds__(256) void resnorm_bwd_kernel(RnParams p) {
    __shared__ float red[8];
    __shared__ float buf[WPR == 1 ? 4 * NV * 256 : 8];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int t = WPR == 1 ? lane : (int)threadIdx.x;
    const float inv = 1.f / (float)p.cols;
    Row<NV> ag1, ab1, ag2, ab2, agt;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) ag1.v[i][j] = ab1.v[i][j] = ag2.v[i][j] = ab2.v[i][j] = agt.v[i][j] = 0.f;
    const int64_t u0 = blockIdx.x * p.per_block, u1 = u0 + p.per_block < p.units ? u0 + p.per_block : p.units;
    for (int64_t u = u0; u < u1; ++u) {
        const int64_t group = u / p.chunks, first = (u % p.chunks) * p.chunk;
        const int64_t last = first + p.chunk < p.each ? first + p.chunk : p.each;
        for (int64_t r = first + (WPR == 1 ? wave : 0); r < last; r += WPR == 1 ? 4 : 1) {
            const int64_t off = (group * p.each + r) * p.cols;
            Row<NV> d, y, k, w;
            rn_load<NV, WPR>(y, p.y, p.y_dt, off, p.cols, p.vec, t);
            if (p.dx_new) rn_load<NV, WPR>(d, p.dx_new, p.x_dt, off, p.cols, p.vec, t);
            else {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) d.v[i][j] = 0.f;
            }
            float mean[2] = {0.f, 0.f}, rstd[2] = {1.f, 1.f};
            if constexpr (PRE) {
                Row<NV> x, dh;
                rn_load<NV, WPR>(x, p.x_new, p.x_dt, off, p.cols, p.vec, t);
                rn_load<NV, WPR>(dh, p.dh, p.h_dt, off, p.cols, p.vec, t);
                rn_load<NV, WPR>(k, p.g2, HH_F32, 0, p.cols, p.vec, t);
                if constexpr (POST) rn_stats2<NV, WPR>(x, y, p.cols, p.rms, p.eps2, p.eps1, t, red, mean, rstd);
                else rn_stats<NV, WPR>(x, p.cols, p.rms, p.eps2, t, red, mean[0], rstd[0]);
                float s[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x.v[i][j] = (x.v[i][j] - mean[0]) * rstd[0];
                        ag2.v[i][j] += dh.v[i][j] * x.v[i][j];
                        ab2.v[i][j] += dh.v[i][j];
                        dh.v[i][j] *= k.v[i][j];
                        s[0] += dh.v[i][j];
                        s[1] += dh.v[i][j] * x.v[i][j];
                    }
                row_sums<2, WPR>(s, red);
                s[0] = p.rms ? 0.f : s[0] * inv;
                s[1] *= inv;
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) d.v[i][j] += rstd[0] * (dh.v[i][j] - s[0] - x.v[i][j] * s[1]);
            } else if constexpr (POST) {
                rn_stats<NV, WPR>(y, p.cols, p.rms, p.eps1, t, red, mean[1], rstd[1]);
            }
            rn_gate<NV, WPR>(w, p, group, t);
            if constexpr (POST) {
                Row<NV> b;
                rn_load<NV, WPR>(k, p.g1, HH_F32, 0, p.cols, p.vec, t);
                if (p.b1) rn_load<NV, WPR>(b, p.b1, HH_F32, 0, p.cols, p.vec, t);
                float s[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool in = rn_in<NV, WPR>(i, j, t, p.cols);
                        const float xh = (y.v[i][j] - mean[1]) * rstd[1];
                        const float dp = in ? d.v[i][j] * w.v[i][j] : 0.f;
                        const float pv = xh * k.v[i][j] + (p.b1 ? b.v[i][j] : 0.f);
                        if (in) agt.v[i][j] += d.v[i][j] * pv;
                        ag1.v[i][j] += dp * xh;
                        ab1.v[i][j] += dp;
                        const float kk = dp * k.v[i][j];
                        s[0] += kk;
                        s[1] += kk * xh;
                        y.v[i][j] = xh;
                        k.v[i][j] = kk;
                    }
                row_sums<2, WPR>(s, red);
                s[0] = p.rms ? 0.f : s[0] * inv;
                s[1] *= inv;
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) y.v[i][j] = rstd[1] * (k.v[i][j] - s[0] - y.v[i][j] * s[1]);
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (rn_in<NV, WPR>(i, j, t, p.cols)) agt.v[i][j] += d.v[i][j] * y.v[i][j];
                        y.v[i][j] = d.v[i][j] * w.v[i][j];
                    }
            }
            rn_store<NV, WPR>(y, p.dy, p.y_dt, off, p.cols, p.vec, t);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) d.v[i][j] *= p.res_scale;
            rn_store<NV, WPR>(d, p.dx, p.x_dt, off, p.cols, p.vec, t);
        }
        if (p.gate_kind != HH_GATE_NONE) {            // a unit's row of gate sums: units never cross groups
            rn_put_cols<NV, WPR>(agt, p.gate_part + u * p.cols, p.cols, t, buf);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) agt.v[i][j] = 0.f;
        }
    }
    const int64_t plane = (int64_t)gridDim.x * p.cols;
    float* out = p.part + blockIdx.x * (int64_t)p.cols;
    if constexpr (POST) {
        rn_put_cols<NV, WPR>(ag1, out, p.cols, t, buf);
        rn_put_cols<NV, WPR>(ab1, out + plane, p.cols, t, buf);
    }
    if constexpr (PRE) {
        rn_put_cols<NV, WPR>(ag2, out + 2 * plane, p.cols, t, buf);
        rn_put_cols<NV, WPR>(ab2, out + 3 * plane, p.cols, t, buf);
    }
}

// out[c] = sum over n rows of part[row][c], rows in order within each of 16 waves and the waves in order: 64 channels to a workgroup.
// blockIdx.y < 4: the norms' planes (out[y] NULL: not wanted); behind them the gate's groups, whose sums take the derivative of tanh
struct RnReduce {
    const float* part; const float* gate_part; const float* gate;
    float* out[4]; float* dgate;
    int64_t blocks, chunks;
    int cols, gate_kind, gate_tanh;
};
__global__ __launch_bounds__(1024) void resnorm_reduce_kernel(RnReduce p) {
    __shared__ float buf[16][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int c = blockIdx.x * 64 + lane;
    const bool is_gate = blockIdx.y >= 4;
    const int64_t group = (int64_t)blockIdx.y - 4;
    float* out = is_gate ? p.dgate : p.out[blockIdx.y];
    if (out == nullptr) return;
    const int64_t n = is_gate ? p.chunks : p.blocks;
    const float* src = is_gate ? p.gate_part + group * p.chunks * p.cols : p.part + blockIdx.y * p.blocks * p.cols;
    const int64_t share = (n + 15) / 16, r0 = wave * share, r1 = r0 + share < n ? r0 + share : n;
    float s = 0.f;
    if (c < p.cols)
        for (int64_t r = r0; r < r1; ++r) s += src[r * p.cols + c];
    buf[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < p.cols) {
        s = 0.f;
#pragma unroll
        for (int w = 0; w < 16; ++w) s += buf[w][lane];
        if (is_gate) {
            const int64_t at = group * p.cols + c;
            if (p.gate_tanh) { const float th = tanhf(p.gate[at]); s *= 1.f - th * th; }
            out[at] = s;
        } else {
            out[c] = s;
        }
    }
}
// scalar gate: all units' rows summed by one workgroup
__global__ __launch_bounds__(1024) void resnorm_scalar_gate_kernel(const float* __restrict__ part, int64_t n, const float* __restrict__ gate, int gate_tanh, float* __restrict__ dgate) {
    __shared__ float buf[16];
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += part[i];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.f;
        for (int w = 0; w < 16; ++w) s += buf[w];
        if (gate_tanh) { const float th = tanhf(gate[0]); s *= 1.f - th * th; }
        dgate[0] = s;
    }
}

// ---- entry points ------------------------------------------------------------------------------------------------------------------------
#define RN_BLOCKS 1024                                // workgroups of the backward pass, about
struct RnPlan { int64_t each, groups, chunk, chunks, units, per_block, blocks; };
static RnPlan rn_plan(int64_t rows, int64_t groups) {
    RnPlan q;
    q.groups = groups;
    q.each = rows / groups;
    int64_t want = (RN_BLOCKS + groups - 1) / groups;                   // units of a group, none below 8 rows unless the group is
    const int64_t most = (q.each + 7) / 8;
    if (want > most) want = most;
    if (want < 1) want = 1;
    q.chunk = (q.each + want - 1) / want;
    q.chunks = (q.each + q.chunk - 1) / q.chunk;
    q.units = q.chunks * groups;
    q.per_block = (q.units + RN_BLOCKS - 1) / RN_BLOCKS;
    q.blocks = (q.units + q.per_block - 1) / q.per_block;
    return q;
}

static int rn_check(const hh_residual_norm* d, bool bwd, const char* who) {
    HH_REQUIRE(d != nullptr, HH_ERR_SHAPE, "%s: NULL description", who);
    HH_REQUIRE(d->rows >= 0 && d->cols > 0 && d->cols <= 4096, HH_ERR_SHAPE, "%s: cols=%d must be in [1, 4096]", who, d->cols);
    HH_REQUIRE(d->gate_kind >= HH_GATE_NONE && d->gate_kind <= HH_GATE_GROUP, HH_ERR_UNSUPPORTED, "%s: unknown gate kind %d", who, d->gate_kind);
    HH_REQUIRE(d->groups >= 1 && d->groups <= 65000 && d->rows % d->groups == 0 && (d->groups == 1 || d->gate_kind == HH_GATE_GROUP), HH_ERR_SHAPE,
               "%s: %lld rows do not split into %lld gate groups (1 without a gate for each group, 65000 at most)", who, (long long)d->rows, (long long)d->groups);
    HH_REQUIRE((d->x_dtype == HH_F32 || d->x_dtype == HH_BF16) && (d->y_dtype == HH_F32 || d->y_dtype == HH_BF16) && (d->h_dtype == HH_F32 || d->h_dtype == HH_BF16), HH_ERR_DTYPE,
               "%s: bad dtype", who);
    if (d->rows == 0) return HH_OK;
    HH_REQUIRE(d->y != nullptr && d->x_new != nullptr && (bwd ? (d->dx != nullptr && d->dy != nullptr) : d->x != nullptr), HH_ERR_ALIGN, "%s: NULL pointer", who);
    HH_REQUIRE((d->gate_kind == HH_GATE_NONE) == (d->gate == nullptr), HH_ERR_ALIGN, "%s: gate kind and pointer do not agree", who);
    HH_REQUIRE(d->post_gamma != nullptr || d->post_beta == nullptr, HH_ERR_ALIGN, "%s: post_beta without post_gamma", who);
    HH_REQUIRE(d->pre_gamma != nullptr || d->pre_beta == nullptr, HH_ERR_ALIGN, "%s: pre_beta without pre_gamma", who);
    if (bwd) HH_REQUIRE((d->dh != nullptr) == (d->pre_gamma != nullptr), HH_ERR_ALIGN, "%s: dh comes with pre_gamma", who);
    else HH_REQUIRE((d->h != nullptr) == (d->pre_gamma != nullptr), HH_ERR_ALIGN, "%s: h comes with pre_gamma", who);
    return HH_OK;
}

static RnParams rn_params(const hh_residual_norm* d) {
    RnParams p;
    p.x = d->x; p.y = d->y; p.x_new = d->x_new; p.h = d->h; p.dx_new = d->dx_new; p.dh = d->dh; p.dx = d->dx; p.dy = d->dy;
    p.gate = d->gate; p.g1 = d->post_gamma; p.b1 = d->post_beta; p.g2 = d->pre_gamma; p.b2 = d->pre_beta;
    p.part = p.gate_part = nullptr;
    p.rows = d->rows; p.each = d->rows / d->groups; p.chunk = p.chunks = p.units = p.per_block = 0;
    p.cols = d->cols; p.gate_kind = d->gate_kind; p.gate_tanh = d->gate_tanh; p.rms = d->rms;
    p.x_dt = d->x_dtype; p.y_dt = d->y_dtype; p.h_dt = d->h_dtype;
    p.eps1 = d->post_eps; p.eps2 = d->pre_eps; p.res_scale = d->res_scale;
    p.vec = d->cols % 4 == 0 && HH_ALIGNED16(p.x) && HH_ALIGNED16(p.y) && HH_ALIGNED16(p.x_new) && HH_ALIGNED16(p.h) && HH_ALIGNED16(p.dx_new) && HH_ALIGNED16(p.dh) && HH_ALIGNED16(p.dx) &&
            HH_ALIGNED16(p.dy) && HH_ALIGNED16(p.gate) && HH_ALIGNED16(p.g1) && HH_ALIGNED16(p.b1) && HH_ALIGNED16(p.g2) && HH_ALIGNED16(p.b2);
    return p;
}

#define RN_DISPATCH(KERNEL, NV, WPR, GRID)                                                                              \
    do {                                                                                                                \
        if (p.g1 && p.g2) hipLaunchKernelGGL((KERNEL<NV, WPR, true, true>), GRID, dim3(256), 0, s, p);                  \
        else if (p.g1) hipLaunchKernelGGL((KERNEL<NV, WPR, true, false>), GRID, dim3(256), 0, s, p);                    \
        else if (p.g2) hipLaunchKernelGGL((KERNEL<NV, WPR, false, true>), GRID, dim3(256), 0, s, p);                    \
        else hipLaunchKernelGGL((KERNEL<NV, WPR, false, false>), GRID, dim3(256), 0, s, p);                             \
    } while (0)
#define RN_BY_COLS(KERNEL, GRID1, GRID4)                                                                                \
    do {                                                                                                                \
        if (p.cols <= 256) RN_DISPATCH(KERNEL, 1, 1, GRID1);                                                            \
        else if (p.cols <= 512) RN_DISPATCH(KERNEL, 2, 1, GRID1);                                                       \
        else if (p.cols <= 768) RN_DISPATCH(KERNEL, 3, 1, GRID1);                                                       \
        else if (p.cols <= 1024) RN_DISPATCH(KERNEL, 4, 1, GRID1);                                                      \
        else if (p.cols <= 2048) RN_DISPATCH(KERNEL, 2, 4, GRID4);                                                      \
        else RN_DISPATCH(KERNEL, 4, 4, GRID4);                                                                          \
    } while (0)

extern "C" int hh_residual_norm_fwd(const hh_residual_norm* d, hh_stream_t stream) {
    const int rc = rn_check(d, false, "hh_residual_norm_fwd");
    if (rc != HH_OK || d->rows == 0) return rc;
    HH_REQUIRE(d->rows <= 0x7fffffff, HH_ERR_SHAPE, "hh_residual_norm_fwd: too many rows");
    hipStream_t s = (hipStream_t)stream;
    const RnParams p = rn_params(d);
    const dim3 by4((unsigned)((d->rows + 3) / 4)), by1((unsigned)d->rows);
    RN_BY_COLS(resnorm_fwd_kernel, by4, by1);
    return hh_check_launch("hh_residual_norm_fwd");
}

extern "C" int64_t hh_workspace_bytes_residual_norm_bwd(int64_t rows, int cols, int64_t groups) {
    if (rows < 0 || cols <= 0 || cols > 4096 || groups < 1 || groups > 65000 || rows % groups) return -1;
    if (rows == 0) return 0;
    const RnPlan q = rn_plan(rows, groups);
    return (4 * q.blocks + q.units) * cols * 4;
}

extern "C" int hh_residual_norm_bwd(const hh_residual_norm* d, hh_stream_t stream) {
    const int rc = rn_check(d, true, "hh_residual_norm_bwd");
    if (rc != HH_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    RnParams p = rn_params(d);
    RnReduce r;
    r.out[0] = d->dpost_gamma; r.out[1] = d->dpost_beta; r.out[2] = d->dpre_gamma; r.out[3] = d->dpre_beta; r.dgate = d->dgate;
    r.part = r.gate_part = nullptr; r.gate = p.gate; r.blocks = r.chunks = 0;
    r.cols = p.cols; r.gate_kind = p.gate_kind; r.gate_tanh = p.gate_tanh;
    HH_REQUIRE((p.gate_kind == HH_GATE_NONE) == (d->dgate == nullptr) && (p.g1 != nullptr) == (d->dpost_gamma != nullptr) && (p.g2 != nullptr) == (d->dpre_gamma != nullptr) &&
                   (p.b1 != nullptr || d->dpost_beta == nullptr) && (p.b2 != nullptr || d->dpre_beta == nullptr),
               HH_ERR_ALIGN, "hh_residual_norm_bwd: a gradient's pointer comes with its parameter's");
    if (d->rows > 0) {
        const RnPlan q = rn_plan(d->rows, d->groups);
        HH_REQUIRE(d->workspace != nullptr && HH_ALIGNED16(d->workspace), HH_ERR_ALIGN, "hh_residual_norm_bwd: a 16-byte aligned workspace is needed");
        p.part = (float*)d->workspace;
        p.gate_part = p.part + 4 * q.blocks * p.cols;
        p.chunk = q.chunk; p.chunks = q.chunks; p.units = q.units; p.per_block = q.per_block;
        r.part = p.part; r.gate_part = p.gate_part; r.blocks = q.blocks; r.chunks = q.chunks;
        const dim3 grid((unsigned)q.blocks);
        RN_BY_COLS(resnorm_bwd_kernel, grid, grid);
    }
    // (no rows: every sum is over nothing, and the launches below write zeros)
    if (p.gate_kind == HH_GATE_SCALAR) {
        hipLaunchKernelGGL(resnorm_scalar_gate_kernel, dim3(1), dim3(1024), 0, s, r.gate_part, d->rows ? r.chunks * p.cols : (int64_t)0, p.gate, p.gate_tanh, d->dgate);
        r.dgate = nullptr;
    }
    if (p.g1 || p.g2 || r.dgate)
        hipLaunchKernelGGL(resnorm_reduce_kernel, dim3((unsigned)((p.cols + 63) / 64), (unsigned)(4 + (r.dgate ? d->groups : 0))), dim3(1024), 0, s, r);
    return hh_check_launch("hh_residual_norm_bwd");
}
