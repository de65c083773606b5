// Weight gradient from an 8-bit activation checkpoint:  dW[m, n] = sum_k dY[k, m] * q[k, n] * s[k, n / 128],  db[m] = sum_k dY[k, m],
// dY bf16 [K tokens, M], q e4m3 [K, N] with a power-of-two scale for 128 channels of a token (act8.hip).
//
// q * s is exact in bf16 (4 significant bits times a power of two), so the operand is turned into bf16 on its way into LDS -- two values an
// instruction, the scale inside it -- and the product runs on v_mfma_f32_16x16x32_bf16 with fp32 sums: the only roundings are those of the sums.
// Both operands stand token-major in memory and in LDS (a row = 128 columns = 256 B); the transposing LDS read delivers the 8 consecutive
// tokens that a lane of the matrix instruction wants.  16-byte chunk c of row r lies at c ^ tn8_key(r), which spreads the four rows x 32 B that
// a 16-lane group reads, and the rows 8 apart of the two groups of a half wave, over the banks.
#include "common.h"

typedef short s16x4_t8 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int tn8_key(int r) { return (2 * (r & 3)) | (((r >> 3) & 1) << 3); }
__device__ __forceinline__ bf16x4 tn8_tr4(const char* addr) {
    s16x4_t8 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t8*)addr);
    return __builtin_bit_cast(bf16x4, r);
}

struct Tn8Params {
    const bf16_t* A; int64_t lda;
    const unsigned char* q; int64_t ldq;
    const float* scale;                    // [K][groups]
    float* C;                              // [splits][M][N]
    float* colsum;                         // [splits][M] or NULL
    int M, N, groups, tiles_n, vec_a, vec_q;
    int64_t K, k_per_split;                // k_per_split: a multiple of 64
};

__global__ __launch_bounds__(256, 2) void gemm_tn8_kernel(Tn8Params p) {
    __shared__ __attribute__((aligned(16))) char smem[2 * 2 * 16384];        // [buffer][A | B][64 rows x 256 B]
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int m0 = (blockIdx.x / p.tiles_n) * 128, n0 = (blockIdx.x % p.tiles_n) * 128;
    const int64_t k0 = (int64_t)blockIdx.y * p.k_per_split;
    const int64_t k1 = k0 + p.k_per_split < p.K ? k0 + p.k_per_split : p.K;
    const int nk = (int)((k1 - k0 + 63) / 64);                                // (0 for a slice behind the last token: zeros are written)

    u32x4 ra[4], rq[2];
    float rs[2];
    auto fetch = [&](int kt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = tid + 256 * i;
            const int64_t k = k0 + (int64_t)kt * 64 + (at >> 4);
            const int m = m0 + (at & 15) * 8;
            ra[i] = (u32x4){0u, 0u, 0u, 0u};
            if (k < k1 && m < p.M) {
                const bf16_t* src = p.A + k * p.lda + m;
                if (p.vec_a) ra[i] = *(const u32x4*)src;
                else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (m + j < p.M) ra[i][j >> 1] |= (unsigned)((const unsigned short*)src)[j] << (16 * (j & 1));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = tid + 256 * i;
            const int64_t k = k0 + (int64_t)kt * 64 + (at >> 3);
            const int n = n0 + (at & 7) * 16;
            rq[i] = (u32x4){0u, 0u, 0u, 0u};
            rs[i] = 1.f;
            if (k < k1 && n < p.N) {
                const unsigned char* src = p.q + k * p.ldq + n;
                if (p.vec_q) rq[i] = *(const u32x4*)src;
                else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (n + j < p.N) rq[i][j >> 2] |= (unsigned)src[j] << (8 * (j & 3));
                }
                rs[i] = p.scale[k * p.groups + n / 128];
            }
        }
    };
    auto put = [&](int buf) {
        char* dA = smem + buf * 32768;
        char* dB = dA + 16384;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = tid + 256 * i, r = at >> 4, c = at & 15;
            *(u32x4*)(dA + r * 256 + ((c ^ tn8_key(r)) << 4)) = ra[i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = tid + 256 * i, r = at >> 3, c = (at & 7) * 2;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 w;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    w[2 * j] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rq[i][2 * h + j], rs[i], false));
                    w[2 * j + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rq[i][2 * h + j], rs[i], true));
                }
                *(u32x4*)(dB + r * 256 + (((c + h) ^ tn8_key(r)) << 4)) = w;
            }
        }
    };
    // 16-lane group g reads tokens 8 g .. 8 g + 7 (+ 32 for the second half of the 64); lane 4 qd + pc of the group gives the address of row qd, columns 4 pc ..
    const int g = lane >> 4, qd = (lane & 15) >> 2, pc = lane & 3;
    auto frag = [&](const char* tile, int col0, int ks) -> bf16x8 {
        const int r0 = 32 * ks + 8 * g + qd, r1 = r0 + 4;
        const int ch = (col0 >> 3) + (pc >> 1);
        const bf16x4 a = tn8_tr4(tile + r0 * 256 + ((ch ^ tn8_key(r0)) << 4) + (pc & 1) * 8);
        const bf16x4 b = tn8_tr4(tile + r1 * 256 + ((ch ^ tn8_key(r1)) << 4) + (pc & 1) * 8);
        return (bf16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    };

    const bool want_cs = p.colsum != nullptr && n0 == 0 && wn == 0;            // db: one more product, against ones
    const bf16x8 ones = {(bf16_t)1.f, (bf16_t)1.f, (bf16_t)1.f, (bf16_t)1.f, (bf16_t)1.f, (bf16_t)1.f, (bf16_t)1.f, (bf16_t)1.f};
    f32x4 cs[4], acc[4][4];                                                    // acc[tn][tm]: rows n, columns m
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        cs[a] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[a][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    if (nk > 0) {
        fetch(0);
        put(0);
    }
    __syncthreads();
    for (int t = 0; t < nk; ++t) {
        const int cur = t & 1;
        if (t + 1 < nk) fetch(t + 1);
        const char* tA = smem + cur * 32768;
        const char* tB = tA + 16384;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            bf16x8 af[4], bf[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                af[i] = frag(tA, wm * 64 + i * 16, ks);
                bf[i] = frag(tB, wn * 64 + i * 16, ks);
            }
#pragma unroll
            for (int tn = 0; tn < 4; ++tn)
#pragma unroll
                for (int tm = 0; tm < 4; ++tm) acc[tn][tm] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[tn], af[tm], acc[tn][tm], 0, 0, 0);
            if (want_cs) {
#pragma unroll
                for (int tm = 0; tm < 4; ++tm) cs[tm] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, af[tm], cs[tm], 0, 0, 0);
            }
        }
        if (t + 1 < nk) put(cur ^ 1);
        __syncthreads();
    }
    const int mr = lane & 15;
    float* Cp = p.C + (int64_t)blockIdx.y * p.M * p.N;
    if (want_cs && g == 0) {
#pragma unroll
        for (int tm = 0; tm < 4; ++tm) {
            const int m = m0 + wm * 64 + tm * 16 + mr;
            if (m < p.M) p.colsum[(int64_t)blockIdx.y * p.M + m] = cs[tm][0];
        }
    }
#pragma unroll
    for (int tm = 0; tm < 4; ++tm) {
        const int m = m0 + wm * 64 + tm * 16 + mr;
        if (m >= p.M) continue;
#pragma unroll
        for (int tn = 0; tn < 4; ++tn) {
            const int n = n0 + wn * 64 + tn * 16 + 4 * g;
            if (n + 4 <= p.N && p.N % 4 == 0) *(f32x4*)(Cp + (int64_t)m * p.N + n) = acc[tn][tm];
            else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + j < p.N) Cp[(int64_t)m * p.N + n + j] = acc[tn][tm][j];
            }
        }
    }
}

// dW and db from the slices' planes, added in slice order
__global__ __launch_bounds__(256) void tn8_join_kernel(const float* __restrict__ part, float* __restrict__ out, int64_t n, const float* __restrict__ cs_part, float* __restrict__ cs, int m,
                                                       int splits) {
    const int64_t total = n + (cs ? m : 0), stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
        const float* src = i < n ? part + i : cs_part + (i - n);
        const int64_t step = i < n ? n : m;
        float a = 0.f;
        for (int s = 0; s < splits; ++s) a += src[s * step];
        if (i < n) out[i] = a;
        else cs[i - n] = a;
    }
}

static int tn8_splits(int M, int N, int64_t K) {
    const int64_t tiles = ((int64_t)(M + 127) / 128) * ((N + 127) / 128);
    int64_t s = 512 / tiles;                                                   // two workgroups to a CU
    const int64_t most = (K + 511) / 512;                                      // and no slice below 512 tokens
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s);
}
static bool tn8_shape_ok(int M, int N, int64_t K) {
    return M > 0 && N > 0 && K >= 0 && M <= (1 << 24) && N <= (1 << 24) && ((int64_t)(M + 127) / 128) * ((N + 127) / 128) <= 0x7fffffff;
}

extern "C" int64_t hh_workspace_bytes_gemm_tn_act8(int M, int N, int64_t K) {
    if (!tn8_shape_ok(M, N, K)) return -1;
    const int64_t s = tn8_splits(M, N, K);
    return s == 1 ? 0 : s * ((int64_t)M * N + M) * 4;
}

extern "C" int hh_gemm_tn_act8(const void* dy, int64_t ld_dy, const void* q, int64_t ldq, const float* scale, float* dw, float* db, int M, int N, int64_t K, void* workspace,
                               hh_stream_t stream) {
    HH_REQUIRE(tn8_shape_ok(M, N, K) && ld_dy >= M && ldq >= N, HH_ERR_SHAPE, "hh_gemm_tn_act8: bad shape (M=%d N=%d K=%lld ld_dy=%lld ldq=%lld)", M, N, (long long)K, (long long)ld_dy, (long long)ldq);
    HH_REQUIRE(dw != nullptr && (K == 0 || (dy != nullptr && q != nullptr && scale != nullptr)), HH_ERR_ALIGN, "hh_gemm_tn_act8: NULL pointer");
    HH_REQUIRE((((uintptr_t)dw) & 15) == 0, HH_ERR_ALIGN, "hh_gemm_tn_act8: dw must be 16-byte aligned");
    const int splits = tn8_splits(M, N, K);
    HH_REQUIRE(splits == 1 || (workspace != nullptr && HH_ALIGNED16(workspace)), HH_ERR_ALIGN, "hh_gemm_tn_act8: a 16-byte aligned workspace is needed");
    hipStream_t s = (hipStream_t)stream;
    Tn8Params p;
    p.A = (const bf16_t*)dy; p.lda = ld_dy; p.q = (const unsigned char*)q; p.ldq = ldq; p.scale = scale;
    p.M = M; p.N = N; p.K = K; p.groups = (N + 127) / 128; p.tiles_n = (N + 127) / 128;
    p.vec_a = M % 8 == 0 && ld_dy % 8 == 0 && HH_ALIGNED16(dy);
    p.vec_q = N % 16 == 0 && ldq % 16 == 0 && HH_ALIGNED16(q);
    p.k_per_split = ((K + 63) / 64 + splits - 1) / splits * 64;
    p.C = splits == 1 ? dw : (float*)workspace;
    p.colsum = db == nullptr ? nullptr : splits == 1 ? db : (float*)workspace + (int64_t)splits * M * N;
    const dim3 grid((unsigned)(((M + 127) / 128) * p.tiles_n), (unsigned)splits);
    hipLaunchKernelGGL(gemm_tn8_kernel, grid, dim3(256), 0, s, p);
    if (splits > 1) {
        const int64_t n = (int64_t)M * N, blocks = (n + M + 255) / 256;
        hipLaunchKernelGGL(tn8_join_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, p.C, dw, n, p.colsum, db, M, splits);
    }
    return hh_check_launch("hh_gemm_tn_act8");
}
