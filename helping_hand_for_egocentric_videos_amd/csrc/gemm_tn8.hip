// Weight gradient from an 8-bit activation checkpoint:  dW[m, n] = sum_k dY[k, m] * q[k, n] * s[k, n / 128],  db[m] = sum_k dY[k, m],
// dY bf16 [K tokens, M], q e4m3 [K, N] with a power-of-two scale for 128 channels of a token (act8.hip).
//
// q * s is exact in bf16 (4 significant bits times a power of two; 2^128 alone is infinite, see act8.hip), so the operand is turned into bf16 on its way into LDS -- two values an
// instruction, the scale inside it -- and the product runs on v_mfma_f32_16x16x32_bf16 with fp32 sums: the only roundings are those of the sums.
// Both operands stand token-major in memory and in LDS (a row = 128 columns = 256 B); the transposing LDS read delivers the 8 consecutive
// tokens that a lane of the matrix instruction wants.  16-byte chunk c of row r lies at c ^ tn8_key(r), which spreads the four rows x 32 B that
// a 16-lane group reads, and the rows 8 apart of the two groups of a half wave, over the banks.
#include "common.h"
#include <type_traits>

typedef short s16x4_t8 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int tn8_key(int r) { return (2 * (r & 3)) | (((r >> 3) & 1) << 3); }
__device__ __forceinline__ bf16x4 tn8_tr4(const char* addr) {
    s16x4_t8 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t8*)addr);
    return __builtin_bit_cast(bf16x4, r);
}

// d += a b.  PIN: in asm, with d in one accumulation register tuple for good -- with 256 accumulators hipcc otherwise permutes them between the products (700 copies in
// the loop, half of its time).  Nothing but these products touches d inside the loop, and two products of one d are WT^2 - 1 others apart.
template <bool PIN>
__device__ __forceinline__ void tn8_mfma(f32x4& d, const bf16x8& a, const bf16x8& b) {
    if constexpr (PIN) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(d) : "v"(a), "v"(b));
    else d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, d, 0, 0, 0);
}

struct Tn8Params {
    const bf16_t* A; int64_t lda;
    const unsigned char* q; int64_t ldq;
    const float* scale;                    // [K][groups]
    float* C;                              // [splits][M][N]
    float* colsum;                         // [splits * db_planes][M] or NULL
    int M, N, groups, tiles_m, tiles_n, splits;
    int db_planes;                         // column tiles that share the tokens of a slice for db
    int64_t K, k_per_split;                // k_per_split: a multiple of the tile's tokens
};

// One tile of the output for one slice of the tokens: 2 x 2 waves of (16 WT) x (16 WT), 32 tokens at a time.
//
// A step is 32 tokens: WT^2 matrix instructions for each wave.  LDS holds four tiles of 32 tokens and the registers are on their way with two more, so that a
// request has two steps' time before its data are put into LDS, and a tile stands there a step before its first fragment is read: one barrier a step.
// WT = 8 (256 x 256, one wave to a SIMD, 256 accumulators): 16 KB of fragments feed 64 instructions of 16 cycles; the four waves' reads take 512 of those
//   1024 cycles of LDS, the writes 256.  Bound by the matrix core and the power that it may draw: 65 552 tokens x 1024 x 4096 with db 449-461 us = 1190-1224 TFLOP/s (442, and
//   13 to join its slices, among 200 passes; 530 among the first twelve, before the clock has settled), where a library product of 8192^3 in bf16 reaches 1263 on the same card,
//   and its product of this shape and layout, from operands that are bf16 already, 818.
// WT = 4 (128 x 128) for outputs and lengths that give the other too few workgroups: bound by a step's latencies (0.3 us with one wave to a SIMD, where its products take
//   0.1), so that two groups of four waves take every second tile each and add their sums at the end (12 320 x 768 x 768 35.9 -> 31.5 us).  A step of both, 64 tokens, takes 0.5 us.
//   A short call is bound by its start and end: of the 16.1 us of 2464 x 768 x 768, five slices of eight steps, the steps are 4.0;  launch, three rounds of loads that wait for each
//   other, the groups' exchange and one slice's store 6.9;  the four more slices, 2.4 MB to write each, 5.2;  and another launch joins them in 4.0.  (768 x 768, one slice: 1 token, four
//   steps with those that fill up, 8.9 us, 512 tokens 10.9;  2, 3, 4, 5 slices of 512 12.9, 14.0, 15.0, 16.1;  seven slices, 7168, 14 336, 28 672 tokens: 19.2, 27.8, 45.2.)
template <int WT, bool VEC>
__global__ __launch_bounds__(WT == 8 ? 256 : 512) void gemm_tn8_kernel(Tn8Params p) {
    constexpr int G = WT == 8 ? 1 : 2;                                                    // groups of four waves: every G-th tile of the slice to each
    constexpr int BLOCK = 32 * WT, BK = 32, ROW = BLOCK * 2, HALF = BK * ROW;     // bytes of a row and of one operand's tile in LDS
    constexpr int CA = BLOCK / 8, CQ = BLOCK / 16;                                       // 16-byte pieces of a row of dY / of q
    constexpr int NA = BK * CA / 256, NQ = BK * CQ / 256, RA = 256 / CA, RQ = 256 / CQ;  // pieces for a thread, rows between them
    constexpr int BUFS = 4;                                                               // tiles in LDS
    extern __shared__ __attribute__((aligned(16))) char smem_all[];                       // [G][BUFS][dY | q][BK][BLOCK] bf16
    const int group = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    char* smem = smem_all + group * BUFS * 2 * HALF;
    const int tid = threadIdx.x & 255, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    // work in the order slice, column tile, row tile; an XCD (blockIdx.x mod 8) takes a contiguous part of it, so that its L2 holds few columns of one slice
    const int total = p.tiles_m * p.tiles_n * p.splits, tiles = p.tiles_m * p.tiles_n;
    const int xcd = blockIdx.x & 7, per = total >> 3, extra = total & 7;
    const int work = xcd * per + (xcd < extra ? xcd : extra) + (blockIdx.x >> 3);
    const int split = work / tiles, tile_n = work % tiles / p.tiles_m, tile_m = work % tiles % p.tiles_m;
    const int m0 = tile_m * BLOCK, n0 = tile_n * BLOCK;
    const int64_t k0 = (int64_t)split * p.k_per_split;
    const int64_t k1 = k0 + p.k_per_split < p.K ? k0 + p.k_per_split : p.K;
    const int nk = k1 > k0 ? (int)((k1 - k0 + G * BK - 1) / (G * BK)) : 0;              // tiles of a group (0 for a slice behind the last token: zeros are written)

    // Buffer loads: a resource ends with the slice, and what lies behind reads as zero -- the rows that fill up the last tile, and the tiles behind it.  Columns behind
    // the last belong to the next row or are zero; their products are not stored.  The resource moves with the tile that is requested, so that offsets stay
    // below 2^31 whatever the slice's length.
    //
    // Any alignment and width (not VEC): the resources begin at a multiple of four bytes at or before the operand and end at one at or behind its end (never in
    // another page than a byte of the operand), a piece is read as the five dwords that hold it and shifted into place; the rows of a thread and its tiles lie a
    // multiple of four bytes apart, so that it has one shift.  Rows behind the last are asked for behind the end, so that they are zeros here too.
    const int ra0 = tid / CA, rq0 = tid / CQ, ca = tid % CA, cq = tid % CQ;
    const unsigned lda = (unsigned)p.lda * 2, ldq = (unsigned)p.ldq, lds = (unsigned)p.groups * 4;      // bytes
    const char* a_at = (const char*)(p.A + k0 * p.lda);
    const char* q_at = (const char*)(p.q + k0 * p.ldq);
    const unsigned a_mis = VEC ? 0 : (unsigned)(uintptr_t)a_at & 3, q_mis = VEC ? 0 : (unsigned)(uintptr_t)q_at & 3;
    const unsigned a_row = a_mis + (unsigned)ra0 * lda, q_row = q_mis + (unsigned)rq0 * ldq;
    const unsigned a_off = a_row + (unsigned)(m0 + ca * 8) * 2, q_off = q_row + (unsigned)(n0 + cq * 16);
    const unsigned s_off = (unsigned)rq0 * lds + (unsigned)((n0 + cq * 16) / 128) * 4;
    struct Stream {
        const char* at; int64_t left; int end;
        __device__ __amdgpu_buffer_rsrc_t next(unsigned bytes) {                          // the resource of this tile; moves on to the next
            end = left < 0 ? 0 : left > 0x7ffffffc ? 0x7ffffffc : (int)left;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, VEC ? end : (end + 3) & ~3, 0x27000);
            at += bytes; left -= bytes;
            return r;
        }
    };
    const int64_t len = k1 - k0;
    Stream a_str = {a_at - a_mis, len * (int64_t)lda + a_mis, 0}, q_str = {q_at - q_mis, len * (int64_t)ldq + q_mis, 0},
           s_str = {(const char*)(p.scale + k0 * p.groups), len * (int64_t)lds, 0};
    // (the last row of a strided operand ends where its columns do, not where a next row would begin)
    a_str.left -= (int64_t)(p.lda - p.M) * 2;
    q_str.left -= p.ldq - p.N;
    if (group) { a_str.next(BK * lda); q_str.next(BK * ldq); s_str.next(BK * lds); }
    struct Regs { u32x4 a[NA], q[NQ]; unsigned a5[VEC ? 1 : NA], q5[VEC ? 1 : NQ]; float s[NQ]; };
    __amdgpu_buffer_rsrc_t a_res, q_res, s_res;
    // piece i of the next tile's rows of dY / of q: pieces in order, tiles in order
    auto fetch_a = [&](int i, Regs& r) {
        if (i == 0) a_res = a_str.next(G * BK * lda);
        const unsigned off = a_off + (unsigned)(RA * i) * lda;
        if constexpr (VEC) r.a[i] = __builtin_amdgcn_raw_buffer_load_b128(a_res, off, 0, 0);
        else {
            const unsigned at = a_row + (unsigned)(RA * i) * lda < (unsigned)a_str.end ? off & ~3u : 0x80000000u;
            r.a[i] = __builtin_amdgcn_raw_buffer_load_b128(a_res, at, 0, 0);
            r.a5[i] = __builtin_amdgcn_raw_buffer_load_b32(a_res, at + 16, 0, 0);
        }
    };
    auto fetch_q = [&](int i, Regs& r) {
        if (i == 0) { q_res = q_str.next(G * BK * ldq); s_res = s_str.next(G * BK * lds); }
        const unsigned off = q_off + (unsigned)(RQ * i) * ldq;
        if constexpr (VEC) r.q[i] = __builtin_amdgcn_raw_buffer_load_b128(q_res, off, 0, 0);
        else {
            const unsigned at = q_row + (unsigned)(RQ * i) * ldq < (unsigned)q_str.end ? off & ~3u : 0x80000000u;
            r.q[i] = __builtin_amdgcn_raw_buffer_load_b128(q_res, at, 0, 0);
            r.q5[i] = __builtin_amdgcn_raw_buffer_load_b32(q_res, at + 16, 0, 0);
        }
        r.s[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(s_res, s_off + (unsigned)(RQ * i) * lds, 0, 0));
    };
    auto shifted = [](const u32x4& v, unsigned v5, unsigned byte) -> u32x4 {             // 16 bytes from byte 0 .. 3 of five dwords
        return (u32x4){__builtin_amdgcn_alignbyte(v[1], v[0], byte), __builtin_amdgcn_alignbyte(v[2], v[1], byte), __builtin_amdgcn_alignbyte(v[3], v[2], byte),
                       __builtin_amdgcn_alignbyte(v5, v[3], byte)};
    };
    float db[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) db[j] = 0.f;
    // db: db_planes of the column tiles share the tokens, each adds up every db_planes-th tile's rows on their way into LDS
    int db_tile = p.colsum != nullptr && tile_n < p.db_planes ? tile_n : -1;
    auto put_a = [&](int t, int i, Regs& r) {
        const int row = ra0 + RA * i;
        if constexpr (!VEC) r.a[i] = shifted(r.a[i], r.a5[i], a_off & 3);
        if (t == db_tile) {
#pragma unroll
            for (int j = 0; j < 4; ++j) { db[2 * j] += bf16_lo_to_f32(r.a[i][j]); db[2 * j + 1] += bf16_hi_to_f32(r.a[i][j]); }
            if (i == NA - 1) db_tile += p.db_planes;
        }
        *(u32x4*)(smem + (t & (BUFS - 1)) * 2 * HALF + row * ROW + ((ca ^ tn8_key(row)) << 4)) = r.a[i];
    };
    auto put_q = [&](int t, int i, int h, Regs& r) {                                // half h of piece i: 8 values, 16 bytes of bf16
        const int row = rq0 + RQ * i;
        if constexpr (!VEC) { if (h == 0) r.q[i] = shifted(r.q[i], r.q5[i], q_off & 3); }
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            w[2 * j] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.q[i][2 * h + j], r.s[i], false));
            w[2 * j + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.q[i][2 * h + j], r.s[i], true));
        }
        *(u32x4*)(smem + (t & (BUFS - 1)) * 2 * HALF + HALF + row * ROW + (((2 * cq + h) ^ tn8_key(row)) << 4)) = w;
    };
    auto fetch = [&](Regs& r) {
#pragma unroll
        for (int i = 0; i < NA; ++i) fetch_a(i, r);
#pragma unroll
        for (int i = 0; i < NQ; ++i) fetch_q(i, r);
    };
    auto put = [&](int t, Regs& r) {
#pragma unroll
        for (int i = 0; i < NA; ++i) put_a(t, i, r);
#pragma unroll
        for (int i = 0; i < NQ; ++i) { put_q(t, i, 0, r); put_q(t, i, 1, r); }
    };
    static_assert(NA + 2 * NQ == WT, "the step below places these pieces");
    // 16-lane group g reads tokens 8 g .. 8 g + 7 of a step; lane 4 qd + pc of the group gives the address of row qd, columns 4 pc .. 4 pc + 3 of 16
    const int g = lane >> 4, qd = (lane & 15) >> 2, pc = lane & 3;
    // rows 4 apart have the same key; piece 2 i + (pc >> 1) of a row lies at 32 (i ^ (key >> 1)) bytes and the low bit: one address for each i
    const int row = 8 * g + qd, key = tn8_key(row) >> 1;
    const int low = row * ROW + ((pc >> 1) << 4) + (pc & 1) * 8;
    int at_a[WT], at_b[WT];
#pragma unroll
    for (int i = 0; i < WT; ++i) {
        const int ia = wm * WT + i, ib = wn * WT + i;
        at_a[i] = low + (((ia & ~7) | ((ia & 7) ^ key)) << 5);
        at_b[i] = low + HALF + (((ib & ~7) | ((ib & 7) ^ key)) << 5);
    }
    auto frag = [&](int at, int buf) -> bf16x8 {
        const char* base = smem + at + (buf & (BUFS - 1)) * 2 * HALF;
        const bf16x4 a = tn8_tr4(base), b = tn8_tr4(base + 4 * ROW);
        return (bf16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    };
    auto frag_a = [&](int buf, int i) { return frag(at_a[i], buf); };
    auto frag_b = [&](int buf, int i) { return frag(at_b[i], buf); };
    f32x4 acc[WT][WT];                                                                    // acc[tn][tm]: rows n, columns m
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < WT; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (nk > 0) {
        Regs r0, r1;
        fetch(r0);
        fetch(r1);
        put(0, r0);
        fetch(r0);
        put(1, r1);
        fetch(r1);
        __syncthreads();
        // fragments: this and the next step's of q, and of dY (WT = 4: a row's four products are shorter than a read's latency) or the next few of it in a ring (WT = 8:
        // there are no registers for two sets, and eight products are longer)
        constexpr bool RING = WT == 8;
        bf16x8 fa[RING ? 4 : 2 * WT], fb[2][WT];
#pragma unroll
        for (int i = 0; i < WT; ++i) {
            fb[0][i] = frag_b(0, i);
            if (!RING || i < 2) fa[i] = frag_a(0, i);
        }
        // One step: the 32 tokens of tile t, P = t mod 4.  The WT^2 matrix instructions go row by row of dY's fragments.  A wave issues in order and a SIMD has
        // one wave (WT = 8), so that everything else is placed between them, an instruction or two behind a product (a product takes 16 cycles): the fragment
        // of dY that is needed two rows (or a step) later, one of the next tile's of q, and the pieces of tile t + 2 that go into LDS with the requests for tile
        // t + 4 that take their registers.  The barrier behind the step shows tile t + 2 to step t + 1, which reads its first fragments; the tile that
        // it replaces, t - 2, was last read before the barrier of step t - 2.
        // The number of steps is rounded up to 4: tiles behind the last are zeros in dY (and what is read ahead of the last step is not used).
        auto step = [&](int t, auto P_) {
            constexpr int P = decltype(P_)::value, cur = P & 1;
            Regs& r = cur ? r1 : r0;
#pragma unroll
            for (int tm = 0; tm < WT; ++tm) {
#pragma unroll
                for (int tn = 0; tn < WT; ++tn) {
                    tn8_mfma<WT == 8>(acc[tn][tm], fb[cur][tn], fa[RING ? tm & 3 : cur * WT + tm]);
                    if (tn == 0) {
                        if (RING) fa[(tm + 2) & 3] = tm + 2 < WT ? frag_a(P, tm + 2) : frag_a(P + 1, tm + 2 - WT);
                        else fa[(cur ^ 1) * WT + tm] = frag_a(P + 1, tm);
                    }
                    if (tn == WT / 4) fb[cur ^ 1][tm] = frag_b(P + 1, tm);
                    if (tn == WT / 2) {
                        if (tm < NA) put_a(t + 2, tm, r);
                        else put_q(t + 2, (tm - NA) / 2, (tm - NA) & 1, r);
                    }
                    if (tn == WT / 2 + WT / 4) {
                        if (tm >= 1 && tm <= NA) fetch_a(tm - 1, r);
                        else if (tm > NA && ((tm - NA) & 1)) fetch_q((tm - NA) / 2, r);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __syncthreads();
        };
        for (int t = 0; t < nk; t += 4) {
            step(t, std::integral_constant<int, 0>());
            step(t + 1, std::integral_constant<int, 1>());
            step(t + 2, std::integral_constant<int, 2>());
            step(t + 3, std::integral_constant<int, 3>());
        }
        if constexpr (WT == 8) {
            // the compiler does not see that these are results of matrix instructions: 16 wait states where 11 are needed before anything else reads one
#pragma unroll
            for (int i = 0; i < WT; ++i)
#pragma unroll
                for (int j = 0; j < WT; ++j) asm volatile("s_nop 15" : "+a"(acc[i][j]));
        }
    }
    if constexpr (G == 2) {
        // the other group's half of the accumulators goes to it through LDS: group 0 ends with the first half of the rows, group 1 with the second
        f32x4* buf = (f32x4*)smem_all + tid;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WT; ++i)
#pragma unroll
            for (int j = 0; j < WT / 2; ++j) buf[((group * WT + i) * (WT / 2) + j) * 256] = group ? acc[i][j] : acc[i][WT / 2 + j];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WT; ++i)
#pragma unroll
            for (int j = 0; j < WT / 2; ++j) {
                const f32x4 other = buf[(((group ^ 1) * WT + i) * (WT / 2) + j) * 256];
                acc[i][j] = group ? acc[i][WT / 2 + j] + other : acc[i][j] + other;      // (the sum of two, the same in either order)
            }
    }
    if (p.colsum != nullptr && tile_n < p.db_planes) {                                                            // the G RA threads of a column, in the order of groups and rows
        float* buf = (float*)smem_all;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) buf[((group * RA + ra0) * CA + ca) * 8 + j] = db[j];
        __syncthreads();
        const int m = m0 + tid;
        if (group == 0 && tid < BLOCK && m < p.M) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < G * RA; ++i) sum += buf[i * BLOCK + tid];
            p.colsum[((int64_t)split * p.db_planes + tile_n) * p.M + m] = sum;
        }
    }
    const int mr = lane & 15;
    float* Cp = p.C + (int64_t)split * p.M * p.N;
#pragma unroll
    for (int tm = 0; tm < WT / G; ++tm) {
        const int m = m0 + wm * 16 * WT + (group * (WT / G) + tm) * 16 + mr;
        if (m >= p.M) continue;
#pragma unroll
        for (int tn = 0; tn < WT; ++tn) {
            const int n = n0 + wn * 16 * WT + tn * 16 + 4 * g;
            if (n + 4 <= p.N) *(f32x4_any*)(Cp + (int64_t)m * p.N + n) = acc[tn][tm];
            else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + j < p.N) Cp[(int64_t)m * p.N + n + j] = acc[tn][tm][j];
            }
        }
    }
}

// dW and db from their planes, added in order: blockIdx.x < blocks: dW, four values to a thread;  behind them 64 channels of db to a workgroup, whose
// waves take a quarter of the planes each
__global__ __launch_bounds__(256) void tn8_join_kernel(const float* __restrict__ part, float* __restrict__ out, int64_t n, int splits, const float* __restrict__ cs_part, float* __restrict__ cs,
                                                       int m, int cs_planes, int blocks) {
    if ((int)blockIdx.x < blocks) {
        const int64_t stride = (int64_t)blocks * 256, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
        for (int64_t i = first; i < n / 4; i += stride) {
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
            for (int s = 0; s < splits; ++s) a += *(const f32x4_any*)(part + s * n + 4 * i);
            *((f32x4*)out + i) = a;
        }
        if (first < n % 4) {
            const int64_t i = n / 4 * 4 + first;
            float a = 0.f;
            for (int s = 0; s < splits; ++s) a += part[s * n + i];
            out[i] = a;
        }
        return;
    }
    __shared__ float buf[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = ((int)blockIdx.x - blocks) * 64 + lane;
    const int share = (cs_planes + 3) / 4, p0 = wave * share, p1 = p0 + share < cs_planes ? p0 + share : cs_planes;
    float a = 0.f;
    if (c < m)
#pragma unroll 8
        for (int s = p0; s < p1; ++s) a += cs_part[(int64_t)s * m + c];
    buf[wave][lane] = a;
    __syncthreads();
    if (wave == 0 && c < m) cs[c] = (buf[0][lane] + buf[1][lane]) + (buf[2][lane] + buf[3][lane]);
}

struct Tn8Plan { int wt, tiles_m, tiles_n, splits, db_planes; };
static Tn8Plan tn8_plan(int M, int N, int64_t K) {
    Tn8Plan q;
    const int64_t large = ((int64_t)(M + 255) / 256) * ((N + 255) / 256);
    // 256 x 256 tiles (one workgroup to a CU) where they nearly fill the chip by themselves (500 x 4096 x 3584: 29.5 us, tiles of 128 45.3; but 2048 x 2560 x 2560, 100
    // of them, 54.2 and 47.3), or with slices of 1024 tokens (65 552 x 1024 x 4096: 465 and 604; 4097 x 2048 x 4096: 85 and 96; 8194 x 1536 x 2048, 432 of
    // them, 69 and 79; 3000 x 2048 x 4096, 384, 71 either way; 4097 x 2048 x 2048, 320, 58 and 48; 12 320 x 768 x 768, 117, 42 and 32)
    q.wt = (large >= 192 || large * ((K + 1023) / 1024) >= 400) && M > 128 && N > 128 ? 8 : 4;
    const int block = 32 * q.wt;
    q.tiles_m = (M + block - 1) / block;
    q.tiles_n = (N + block - 1) / block;
    const int64_t tiles = (int64_t)q.tiles_m * q.tiles_n;
    int64_t s = 256 / tiles;
    // no slice below 512 tokens: every slice leaves a plane of dW to write and to add (2464 x 768 x 768: slices of 352 tokens 20.6 us, 512 19.4, 832 20.9)
    const int64_t most = (K + 511) / 512;
    if (s > most) s = most;
    q.splits = (int)(s < 1 ? 1 : s);
    // one short slice: nothing is left to join, and the workgroups of the first column tile write db (500 x 1024 x 4096 18.4 -> 15.9 us); in a long one the others would
    // wait for them (4096 x 4096 x 4096 134 us either way, 16 384 x 4096 x 4096 shared 442 us, 470 not)
    q.db_planes = q.splits == 1 && K <= 4096 ? 1 : q.tiles_n;
    return q;
}
static bool tn8_shape_ok(int M, int N, int64_t K) {
    return M > 0 && N > 0 && K >= 0 && K <= (1 << 30) && M <= (1 << 24) && N <= (1 << 24) && ((int64_t)(M + 127) / 128) * ((N + 127) / 128) <= (1 << 24);
}

extern "C" int64_t hh_workspace_bytes_gemm_tn_act8(int M, int N, int64_t K) {
    if (!tn8_shape_ok(M, N, K)) return -1;
    const Tn8Plan q = tn8_plan(M, N, K);
    const int64_t db = (int64_t)q.splits * q.db_planes * M;
    if (q.splits == 1) return q.db_planes == 1 ? 0 : db * 4;
    return (((int64_t)q.splits * M * N + 3) / 4 * 4 + db) * 4;
}

extern "C" int hh_gemm_tn_act8(const void* dy, int64_t ld_dy, const void* q, int64_t ldq, const float* scale, float* dw, float* db, int M, int N, int64_t K, void* workspace,
                               hh_stream_t stream) {
    HH_REQUIRE(tn8_shape_ok(M, N, K) && ld_dy >= M && ldq >= N, HH_ERR_SHAPE, "hh_gemm_tn_act8: bad shape (M=%d N=%d K=%lld ld_dy=%lld ldq=%lld)", M, N, (long long)K, (long long)ld_dy, (long long)ldq);
    HH_REQUIRE(ld_dy <= (1 << 24) && ldq <= (1 << 24), HH_ERR_SHAPE, "hh_gemm_tn_act8: leading dimensions up to 2^24");
    HH_REQUIRE(dw != nullptr && (K == 0 || (dy != nullptr && q != nullptr && scale != nullptr)), HH_ERR_ALIGN, "hh_gemm_tn_act8: NULL pointer");
    HH_REQUIRE((((uintptr_t)dw) & 15) == 0, HH_ERR_ALIGN, "hh_gemm_tn_act8: dw must be 16-byte aligned");
    const Tn8Plan pl = tn8_plan(M, N, K);
    const bool joined = pl.splits > 1 || (db != nullptr && pl.db_planes > 1);
    HH_REQUIRE(!joined || (workspace != nullptr && HH_ALIGNED16(workspace)), HH_ERR_ALIGN, "hh_gemm_tn_act8: a 16-byte aligned workspace is needed");
    hipStream_t s = (hipStream_t)stream;
    const int64_t n = (int64_t)M * N;
    Tn8Params p;
    p.A = (const bf16_t*)dy; p.lda = ld_dy; p.q = (const unsigned char*)q; p.ldq = ldq; p.scale = scale;
    p.M = M; p.N = N; p.K = K; p.groups = (N + 127) / 128; p.tiles_m = pl.tiles_m; p.tiles_n = pl.tiles_n; p.splits = pl.splits;
    const int tokens = pl.wt == 8 ? 32 : 64;                                    // (a tile for each group)
    p.k_per_split = ((K + tokens - 1) / tokens + pl.splits - 1) / pl.splits * tokens;
    p.C = pl.splits == 1 ? dw : (float*)workspace;
    p.db_planes = pl.db_planes;
    p.colsum = db == nullptr ? nullptr : !joined ? db : (float*)workspace + (pl.splits == 1 ? 0 : (n * pl.splits + 3) / 4 * 4);
    const bool vec = M % 8 == 0 && ld_dy % 8 == 0 && HH_ALIGNED16(dy) && N % 16 == 0 && ldq % 16 == 0 && HH_ALIGNED16(q);
    const dim3 grid((unsigned)(pl.tiles_m * pl.tiles_n * pl.splits));
    const int lds = 128 * 1024;
    {
        static std::atomic<uint64_t> attr{0};
        if (hh_attr_needed(attr)) {
            hipError_t e = hipFuncSetAttribute((const void*)gemm_tn8_kernel<8, true>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            if (e == hipSuccess) e = hipFuncSetAttribute((const void*)gemm_tn8_kernel<8, false>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            if (e == hipSuccess) e = hipFuncSetAttribute((const void*)gemm_tn8_kernel<4, true>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            if (e == hipSuccess) e = hipFuncSetAttribute((const void*)gemm_tn8_kernel<4, false>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            HH_REQUIRE(e == hipSuccess, HH_ERR_LAUNCH, "hh_gemm_tn_act8: %s", hipGetErrorString(e));
            hh_attr_done(attr);
        }
    }
    if (pl.wt == 8) {
        if (vec) hipLaunchKernelGGL((gemm_tn8_kernel<8, true>), grid, dim3(256), lds, s, p);
        else hipLaunchKernelGGL((gemm_tn8_kernel<8, false>), grid, dim3(256), lds, s, p);
    } else {
        if (vec) hipLaunchKernelGGL((gemm_tn8_kernel<4, true>), grid, dim3(512), lds, s, p);
        else hipLaunchKernelGGL((gemm_tn8_kernel<4, false>), grid, dim3(512), lds, s, p);
    }
    if (joined) {
        int64_t blocks = pl.splits == 1 ? 0 : (n / 4 + 255) / 256;
        if (pl.splits > 1) blocks = blocks < 1 ? 1 : blocks > 4096 ? 4096 : blocks;
        hipLaunchKernelGGL(tn8_join_kernel, dim3((unsigned)(blocks + (db ? (M + 63) / 64 : 0))), dim3(256), 0, s, p.C, dw, n, pl.splits, p.colsum, db, M, pl.splits * pl.db_planes, (int)blocks);
    }
    return hh_check_launch("hh_gemm_tn_act8");
}
