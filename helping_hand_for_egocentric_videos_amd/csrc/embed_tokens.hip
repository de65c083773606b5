// Token embedding:  out[s, t, :] = scale * W[id[s, t], :] + pos[t, :]   (CLIP.encode_text, model/LaviLa.py:660-663), and its gradients
//     dW[v, :] = scale * sum_{id[s, t] = v} dy[s, t, :],   dpos[t, :] = sum_s dy[s, t, :].
//
// The gradient goes by SORTED tokens: a stable radix sort of the ids (whole numbers only) puts the positions of one row next to each other, in
// ascending order; the sorted list is cut into chunks, a workgroup sums the runs of equal ids of its chunk in registers (fp32), writes the runs
// that lie inside the chunk to dW and leaves the sums of runs that cross a border in the workspace; a second launch joins those in chunk order.
// No floating-point atomics: the order of every sum depends on the ids alone, so that equal inputs give equal bits, and a row named by most
// of the tokens (padding, start and end marks) is summed by as many workgroups as its share of the list.
#include "common.h"

typedef unsigned int u32;

// ---- forward ---------------------------------------------------------------------------------------------------------------------------
template <int E> struct fvec { float v[E]; };

// E consecutive elements as fp32; `whole`: the address is aligned for one wide access and all E exist, else `n` of them one by one
template <int E, typename T>
__device__ __forceinline__ fvec<E> load_e(const T* p, bool whole, int n) {
    fvec<E> r;
    if (whole) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const f32x4 t = *(const f32x4*)(p + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) r.v[i + j] = t[j];
            }
        } else if constexpr (E == 8) {
            const u32x4 t = *(const u32x4*)p;
#pragma unroll
            for (int j = 0; j < 4; ++j) { r.v[2 * j] = bf16_lo_to_f32(t[j]); r.v[2 * j + 1] = bf16_hi_to_f32(t[j]); }
        } else {
            const u32x2 t = *(const u32x2*)p;
#pragma unroll
            for (int j = 0; j < 2; ++j) { r.v[2 * j] = bf16_lo_to_f32(t[j]); r.v[2 * j + 1] = bf16_hi_to_f32(t[j]); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) r.v[i] = i < n ? (float)p[i] : 0.f;
    }
    return r;
}
template <int E, typename T>
__device__ __forceinline__ void store_e(T* p, const fvec<E>& r, bool whole, int n) {
    if (whole) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < E; i += 4) { f32x4 t = {r.v[i], r.v[i + 1], r.v[i + 2], r.v[i + 3]}; *(f32x4*)(p + i) = t; }
        } else if constexpr (E == 8) {
            u32x4 t = {pack_bf16(r.v[0], r.v[1]), pack_bf16(r.v[2], r.v[3]), pack_bf16(r.v[4], r.v[5]), pack_bf16(r.v[6], r.v[7])};
            *(u32x4*)p = t;
        } else {
            u32x2 t = {pack_bf16(r.v[0], r.v[1]), pack_bf16(r.v[2], r.v[3])};
            *(u32x2*)p = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < n) p[i] = (T)r.v[i];
    }
}

__device__ __forceinline__ int64_t load_id(const void* ids, int wide, int64_t i) {
    return wide ? ((const int64_t*)ids)[i] : (int64_t)((const int*)ids)[i];
}

// lpr lanes (a power of two) share a row, each takes every lpr-th piece of E elements; 64 / lpr rows to a wave
template <typename TW, typename TO, int E>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* __restrict__ ids, int wide, const TW* __restrict__ w, const float* __restrict__ pos, TO* __restrict__ out,
                                                        int64_t n, int length, int64_t rows, int dim, float scale, int lpr_log2, int aligned) {
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t r = (wave << (6 - lpr_log2)) + (lane >> lpr_log2);
    if (r >= n) return;
    const int64_t id = load_id(ids, wide, r);
    const bool known = id >= 0 && id < rows;
    const TW* wr = w + (known ? id : 0) * dim;
    const float* pr = pos ? pos + (r % length) * (int64_t)dim : nullptr;
    TO* o = out + r * dim;
    for (int c = (lane & ((1 << lpr_log2) - 1)) * E; c < dim; c += E << lpr_log2) {
        const bool whole = aligned && c + E <= dim;
        fvec<E> v;
        if (known) {
            v = load_e<E, TW>(wr + c, whole, dim - c);
            if (pr) {
                const fvec<E> p = load_e<E, float>(pr + c, whole, dim - c);
#pragma unroll
                for (int i = 0; i < E; ++i) v.v[i] = v.v[i] * scale + p.v[i];
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) v.v[i] *= scale;
            }
        } else {                                     // an id without a row shows in the result (there is no error to return from a launch)
#pragma unroll
            for (int i = 0; i < E; ++i) v.v[i] = __builtin_nanf("");
        }
        store_e<E, TO>(o + c, v, whole, dim - c);
    }
}

// ---- the sort: least significant digit first, stable, two launches for each digit --------------------------------------------------------
#define SORT_BLOCKS 256                              // at most: a block's share of the list grows with it

struct SortPass { int shift, bits; };
struct SortPlan { int blocks, per_block, passes; SortPass pass[4]; };

static SortPlan sort_plan(int64_t n, int64_t rows) {
    SortPlan p;
    p.blocks = (int)((n + 1023) / 1024);
    if (p.blocks > SORT_BLOCKS) p.blocks = SORT_BLOCKS;
    if (p.blocks < 1) p.blocks = 1;
    p.per_block = (int)(((n + p.blocks - 1) / p.blocks + 255) / 256 * 256);
    int bits = 1;
    while ((rows >> bits) != 0) ++bits;              // keys 0 .. rows (rows = "no row")
    p.passes = (bits + 7) / 8;
    for (int i = 0, at = 0; i < p.passes; ++i) {
        const int b = (bits - at + p.passes - i - 1) / (p.passes - i);
        p.pass[i].shift = at;
        p.pass[i].bits = b;
        at += b;
    }
    return p;
}

// counts of one digit in a block's share; the first pass also turns ids into keys (no row: `rows`, which sorts behind all others)
__global__ __launch_bounds__(256) void sort_count_kernel(const void* __restrict__ ids, int wide, int64_t rows, int64_t skip, u32* __restrict__ keys, u32* __restrict__ hist, int n,
                                                         int per_block, int shift, int bits) {
    __shared__ u32 count[256];
    count[threadIdx.x] = 0;
    __syncthreads();
    const int64_t b0 = (int64_t)blockIdx.x * per_block;
    const int64_t b1 = b0 + per_block < n ? b0 + per_block : n;
    for (int64_t i = b0 + threadIdx.x; i < b1; i += 256) {
        u32 key;
        if (ids) {
            const int64_t id = load_id(ids, wide, i);
            key = id >= 0 && id < rows && id != skip ? (u32)id : (u32)rows;
            keys[i] = key;
        } else {
            key = keys[i];
        }
        atomicAdd(&count[(key >> shift) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    hist[(int64_t)blockIdx.x * 256 + threadIdx.x] = count[threadIdx.x];
}

// places a block's share behind the smaller digits and behind the earlier blocks' equal ones; `from`: NULL on the first pass (position i)
__global__ __launch_bounds__(256) void sort_place_kernel(const u32* __restrict__ keys, const u32* __restrict__ from, const u32* __restrict__ hist, u32* __restrict__ keys_out,
                                                         u32* __restrict__ from_out, int n, int per_block, int shift, int bits) {
    __shared__ u32 base[256], wcount[4][256], part[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    u32 before = 0, total = 0;
    for (int b = 0; b < (int)gridDim.x; ++b) {
        const u32 h = hist[(int64_t)b * 256 + tid];
        if (b < (int)blockIdx.x) before += h;
        total += h;
    }
    u32 incl = total;                                // digits below `tid`: inclusive scan over the wave, then over the four waves
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u32 t = __shfl_up(incl, o, 64);
        if (lane >= o) incl += t;
    }
    if (lane == 63) part[wave] = incl;
    __syncthreads();
    for (int w = 0; w < wave; ++w) incl += part[w];
    base[tid] = incl - total + before;
    const int64_t b0 = (int64_t)blockIdx.x * per_block;
    const int64_t b1 = b0 + per_block < n ? b0 + per_block : n;
    for (int64_t r = b0; r < b1; r += 256) {
#pragma unroll
        for (int w = 0; w < 4; ++w) wcount[w][tid] = 0;
        __syncthreads();
        const int64_t i = r + tid;
        const bool valid = i < b1;
        const u32 key = valid ? keys[i] : 0;
        const u32 digit = (key >> shift) & ((1u << bits) - 1);
        uint64_t same = __ballot(valid);             // lanes of this wave with the same digit
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((digit >> b) & 1);
            same &= ((digit >> b) & 1) ? set : ~set;
        }
        const u32 rank = (u32)__popcll(same & ((1ull << lane) - 1));
        if (valid && rank == 0) wcount[wave][digit] = (u32)__popcll(same);
        __syncthreads();
        if (valid) {
            u32 at = base[digit] + rank;
            for (int w = 0; w < wave; ++w) at += wcount[w][digit];
            keys_out[at] = key;
            from_out[at] = from ? from[i] : (u32)i;
        }
        __syncthreads();
        base[tid] += wcount[0][tid] + wcount[1][tid] + wcount[2][tid] + wcount[3][tid];
    }
}

// ---- the sums over runs of equal keys ----------------------------------------------------------------------------------------------------
struct RunParams {
    const u32* keys; const u32* from;                // sorted keys and the positions they came from; keys == NULL: the list of dpos, see run_key
    const void* dy;
    float* out;                                      // [rows, dim]
    float* part;                                     // [chunks][2][dim]: a chunk's first run where it began earlier, its last where it goes on
    int n, chunk, dim, accumulate, aligned;
    int length, seqs;                                // dpos: entry j is row t = j / seqs of the sequence j % seqs
    int64_t rows;
    float scale;
};
__device__ __forceinline__ u32 run_key(const RunParams& p, int j) { return p.keys ? p.keys[j] : (u32)(j / p.seqs); }
__device__ __forceinline__ int64_t run_from(const RunParams& p, int j) { return p.keys ? (int64_t)p.from[j] : (int64_t)(j % p.seqs) * p.length + j / p.seqs; }

__device__ __forceinline__ void put_row(const RunParams& p, u32 key, int c, bool whole, fvec<4> v) {
    float* o = p.out + (int64_t)key * p.dim + c;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.v[i] *= p.scale;
    if (p.accumulate) {
        const fvec<4> t = load_e<4, float>(o, whole, p.dim - c);
#pragma unroll
        for (int i = 0; i < 4; ++i) v.v[i] += t.v[i];
    }
    store_e<4, float>(o, v, whole, p.dim - c);
}

template <typename T>
__global__ __launch_bounds__(256) void run_sum_kernel(RunParams p) {
    const int c = (blockIdx.y * 256 + threadIdx.x) * 4;
    if (c >= p.dim) return;
    const bool whole = p.aligned && c + 4 <= p.dim;
    const int j0 = blockIdx.x * p.chunk, j1 = j0 + p.chunk < p.n ? j0 + p.chunk : p.n;
    u32 key = run_key(p, j0);
    bool head = j0 > 0 && run_key(p, j0 - 1) == key;  // this run began in an earlier chunk
    fvec<4> acc = {{0.f, 0.f, 0.f, 0.f}};
    for (int j = j0; j < j1 && (int64_t)key < p.rows; ++j) {
        const fvec<4> v = load_e<4, T>((const T*)p.dy + run_from(p, j) * p.dim + c, whole, p.dim - c);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc.v[i] += v.v[i];
        const bool last = j + 1 == p.n;
        const u32 next = last ? 0 : run_key(p, j + 1);
        if (!last && next == key && j + 1 < j1) continue;
        const bool goes_on = !last && next == key;
        if (head) store_e<4, float>(p.part + ((int64_t)blockIdx.x * 2) * p.dim + c, acc, whole, p.dim - c);
        else if (goes_on) store_e<4, float>(p.part + ((int64_t)blockIdx.x * 2 + 1) * p.dim + c, acc, whole, p.dim - c);
        else put_row(p, key, c, whole, acc);
        acc = fvec<4>{{0.f, 0.f, 0.f, 0.f}};
        head = false;
        if (!last) key = next;
    }
}

// a run that starts in chunk b and goes on: its part of chunk b and of the chunks behind, added in that order
__global__ __launch_bounds__(256) void run_join_kernel(RunParams p) {
    const int c = (blockIdx.y * 256 + threadIdx.x) * 4;
    const int b = blockIdx.x;
    const int j1 = (b + 1) * p.chunk;
    if (c >= p.dim || j1 >= p.n) return;
    const u32 key = run_key(p, j1);
    if ((int64_t)key >= p.rows || run_key(p, j1 - 1) != key) return;           // nothing crosses this border
    const int j0 = b * p.chunk;
    if (j0 > 0 && run_key(p, j0) == key && run_key(p, j0 - 1) == key) return;   // it began before this chunk
    const bool whole = p.aligned && c + 4 <= p.dim;
    fvec<4> acc = load_e<4, float>(p.part + ((int64_t)b * 2 + 1) * p.dim + c, whole, p.dim - c);
    for (int k = b + 1; (int64_t)k * p.chunk < p.n && run_key(p, k * p.chunk) == key; ++k) {
        const fvec<4> v = load_e<4, float>(p.part + ((int64_t)k * 2) * p.dim + c, whole, p.dim - c);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc.v[i] += v.v[i];
    }
    put_row(p, key, c, whole, acc);
}

__global__ __launch_bounds__(256) void fill_zero_kernel(float* __restrict__ p, int64_t n) {
    const int64_t stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) p[i] = 0.f;
}

static int run_chunk(int64_t n) {
    int64_t c = (n + 2047) / 2048;                   // about 2048 workgroups for a long list, and at least 32 rows for each
    return (int)(c < 32 ? 32 : c);
}
static int64_t run_chunks(int64_t n) { return n ? (n + run_chunk(n) - 1) / run_chunk(n) : 0; }

// ---- entry points ------------------------------------------------------------------------------------------------------------------------
static bool embed_shape_ok(int64_t seqs, int length, int64_t rows, int dim) {
    return seqs >= 0 && length > 0 && rows > 0 && rows < 0x7fffffff && dim > 0 && dim <= (1 << 20) && seqs * (double)length < 1073741824.0;
}

extern "C" int hh_embed_tokens_fwd(const void* ids, int id_bytes, const void* weight, int w_dtype, const float* pos, void* out, int out_dtype, int64_t seqs, int length, int64_t rows,
                                   int dim, float scale, hh_stream_t stream) {
    HH_REQUIRE(embed_shape_ok(seqs, length, rows, dim), HH_ERR_SHAPE, "hh_embed_tokens_fwd: need length, rows, dim > 0, dim <= 2^20 and fewer than 2^30 tokens and 2^31 rows (seqs=%lld length=%d rows=%lld dim=%d)",
               (long long)seqs, length, (long long)rows, dim);
    HH_REQUIRE(id_bytes == 4 || id_bytes == 8, HH_ERR_DTYPE, "hh_embed_tokens_fwd: ids are 4 or 8 bytes wide");
    HH_REQUIRE((w_dtype == HH_F32 || w_dtype == HH_BF16) && (out_dtype == HH_F32 || out_dtype == HH_BF16), HH_ERR_DTYPE, "hh_embed_tokens_fwd: bad dtype");
    const int64_t n = seqs * length;
    if (n == 0) return HH_OK;
    HH_REQUIRE(ids != nullptr && weight != nullptr && out != nullptr, HH_ERR_ALIGN, "hh_embed_tokens_fwd: NULL pointer");
    hipStream_t s = (hipStream_t)stream;
    const bool al = HH_ALIGNED16(weight) && HH_ALIGNED16(out) && HH_ALIGNED16(pos);
#define EF(TW, TO, E)                                                                                                                            \
    do {                                                                                                                                         \
        int l = 0;                                                                                                                               \
        while (l < 6 && ((int64_t)E << l) < dim) ++l;                                                                                            \
        const int64_t waves = (n + (64 >> l) - 1) / (64 >> l), blocks = (waves + 3) / 4;                                                         \
        hipLaunchKernelGGL((embed_fwd_kernel<TW, TO, E>), dim3((unsigned)blocks), dim3(256), 0, s, ids, id_bytes == 8, (const TW*)weight, pos, (TO*)out, n, length, rows, dim, scale, l, \
                           (int)(al && dim % E == 0));                                                                                           \
    } while (0)
    if (w_dtype == HH_F32 && out_dtype == HH_F32) EF(float, float, 4);
    else if (w_dtype == HH_F32) EF(float, bf16_t, 4);
    else if (out_dtype == HH_F32) EF(bf16_t, float, 4);
    else EF(bf16_t, bf16_t, 8);
#undef EF
    return hh_check_launch("hh_embed_tokens_fwd");
}

static int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

extern "C" int64_t hh_workspace_bytes_embed_tokens_bwd(int64_t seqs, int length, int64_t rows, int dim) {
    if (!embed_shape_ok(seqs, length, rows, dim)) return -1;
    const int64_t n = seqs * length;
    return 4 * align256(4 * n) + align256(SORT_BLOCKS * 256 * 4) + align256(run_chunks(n) * 2 * (int64_t)dim * 4);
}

extern "C" int hh_embed_tokens_bwd(const void* ids, int id_bytes, const void* dy, int dy_dtype, float* dweight, int accumulate, float* dpos, int64_t seqs, int length, int64_t rows,
                                   int dim, float scale, int64_t skip_id, void* workspace, hh_stream_t stream) {
    HH_REQUIRE(embed_shape_ok(seqs, length, rows, dim), HH_ERR_SHAPE, "hh_embed_tokens_bwd: need length, rows, dim > 0, dim <= 2^20 and fewer than 2^30 tokens and 2^31 rows (seqs=%lld length=%d rows=%lld dim=%d)",
               (long long)seqs, length, (long long)rows, dim);
    HH_REQUIRE(id_bytes == 4 || id_bytes == 8, HH_ERR_DTYPE, "hh_embed_tokens_bwd: ids are 4 or 8 bytes wide");
    HH_REQUIRE(dy_dtype == HH_F32 || dy_dtype == HH_BF16, HH_ERR_DTYPE, "hh_embed_tokens_bwd: bad dtype");
    HH_REQUIRE(dweight != nullptr, HH_ERR_ALIGN, "hh_embed_tokens_bwd: dweight is NULL");
    hipStream_t s = (hipStream_t)stream;
    const int64_t n = seqs * length;
    HH_REQUIRE(n == 0 || (ids != nullptr && dy != nullptr && workspace != nullptr && HH_ALIGNED16(workspace)), HH_ERR_ALIGN,
               "hh_embed_tokens_bwd: ids, dy and a 16-byte aligned workspace are needed");
    if (!accumulate) {
        const int64_t total = rows * dim, blocks = (total + 1023) / 1024;
        hipLaunchKernelGGL(fill_zero_kernel, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, s, dweight, total);
    }
    if (n == 0) {
        if (dpos) hipLaunchKernelGGL(fill_zero_kernel, dim3(64), dim3(256), 0, s, dpos, (int64_t)length * dim);
        return hh_check_launch("hh_embed_tokens_bwd");
    }
    char* ws = (char*)workspace;
    u32* keys[2] = {(u32*)ws, (u32*)(ws + align256(4 * n))};
    u32* from[2] = {(u32*)(ws + 2 * align256(4 * n)), (u32*)(ws + 3 * align256(4 * n))};
    u32* hist = (u32*)(ws + 4 * align256(4 * n));
    float* part = (float*)(ws + 4 * align256(4 * n) + align256(SORT_BLOCKS * 256 * 4));
    const SortPlan sp = sort_plan(n, rows);
    for (int i = 0; i < sp.passes; ++i) {
        hipLaunchKernelGGL(sort_count_kernel, dim3(sp.blocks), dim3(256), 0, s, i == 0 ? ids : nullptr, id_bytes == 8, rows, skip_id, keys[i & 1], hist, (int)n, sp.per_block,
                           sp.pass[i].shift, sp.pass[i].bits);
        hipLaunchKernelGGL(sort_place_kernel, dim3(sp.blocks), dim3(256), 0, s, keys[i & 1], i == 0 ? nullptr : from[i & 1], hist, keys[(i + 1) & 1], from[(i + 1) & 1], (int)n,
                           sp.per_block, sp.pass[i].shift, sp.pass[i].bits);
    }
    RunParams p;
    p.keys = keys[sp.passes & 1]; p.from = from[sp.passes & 1];
    p.dy = dy; p.out = dweight; p.part = part;
    p.n = (int)n; p.chunk = run_chunk(n); p.dim = dim; p.accumulate = accumulate != 0;
    p.aligned = dim % 4 == 0 && HH_ALIGNED16(dy) && HH_ALIGNED16(dweight);
    p.length = length; p.seqs = (int)seqs; p.rows = rows; p.scale = scale;
    const int need = (dim + 3) / 4;
    const int threads = need >= 256 ? 256 : (need + 63) / 64 * 64;
    const dim3 grid((unsigned)run_chunks(n), (unsigned)((need + 255) / 256));
    for (int which = 0; which < 2; ++which) {
        if (which == 1) {
            if (!dpos) break;
            p.keys = p.from = nullptr;
            p.out = dpos; p.accumulate = 0; p.scale = 1.f; p.rows = length;
            p.aligned = dim % 4 == 0 && HH_ALIGNED16(dy) && HH_ALIGNED16(dpos);
        }
        if (dy_dtype == HH_F32) hipLaunchKernelGGL(run_sum_kernel<float>, grid, dim3(threads), 0, s, p);
        else hipLaunchKernelGGL(run_sum_kernel<bf16_t>, grid, dim3(threads), 0, s, p);
        hipLaunchKernelGGL(run_join_kernel, grid, dim3(threads), 0, s, p);
    }
    return hh_check_launch("hh_embed_tokens_bwd");
}
