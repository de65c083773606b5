// Token embedding:  out[s, t, :] = scale * W[id[s, t], :] + pos[t, :]   (CLIP.encode_text, model/LaviLa.py:660-663), and its gradients
//     dW[v, :] = scale * sum_{id[s, t] = v} dy[s, t, :],   dpos[t, :] = sum_s dy[s, t, :].
//
// The gradient goes by SORTED tokens: a stable radix sort of the ids (whole numbers only) puts the positions of one row next to each other, in
// ascending order; the sorted list is cut into chunks, a workgroup sums the runs of equal ids of its chunk in registers (fp32), writes the runs
// that lie inside the chunk to dW and leaves the sums of runs that cross a border in the workspace; a second launch joins those in chunk order.
// No floating-point atomics: the order of every sum depends on the ids alone, so that equal inputs give equal bits, and a row named by most
// of the tokens (padding, start and end marks) is summed by as many workgroups as its share of the list.  Up to 512 or 1024 tokens need no list at all (direct_kernel).
//
// Measured:  forward 2048 x 77 of 768 fp32 with pos 81 us, 6.6 TB/s, bound by the writes (a fill: 6.8).  Gradient 160 x 77 of 49 408 x 768 fp32 with dpos 58 us: four
// launches of 7 us that sort and, for the most of their time, fill dweight with zeros (152 MB), 20 us of sums (dy read twice, the second time from the cache), 12 us
// for the runs that cross chunks.  64 x 2048 of 49 408 x 1024 bf16 142 us, nearly all of it the sums (rows gathered, 2 KB
// each, at 4.2 TB/s) with the zeros of the rows that no id names.
#include "common.h"

typedef unsigned int u32;

// ---- forward ---------------------------------------------------------------------------------------------------------------------------
template <int E> struct fvec { float v[E]; };

// E consecutive elements as fp32, in wide accesses where all E exist (`whole`), else `n` of them one by one
template <int E, typename T>
__device__ __forceinline__ fvec<E> load_e(const T* p, bool whole, int n) {
    fvec<E> r;
    if (whole) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const f32x4 t = *(const f32x4_any*)(p + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) r.v[i + j] = t[j];
            }
        } else if constexpr (E == 8) {
            const u32x4 t = *(const u32x4_any*)p;
#pragma unroll
            for (int j = 0; j < 4; ++j) { r.v[2 * j] = bf16_lo_to_f32(t[j]); r.v[2 * j + 1] = bf16_hi_to_f32(t[j]); }
        } else {
            const u32x2 t = *(const u32x2_any*)p;
#pragma unroll
            for (int j = 0; j < 2; ++j) { r.v[2 * j] = bf16_lo_to_f32(t[j]); r.v[2 * j + 1] = bf16_hi_to_f32(t[j]); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) r.v[i] = i < n ? (float)p[i] : 0.f;
    }
    return r;
}
template <int E, typename T, bool NT = false>
__device__ __forceinline__ void store_e(T* p, const fvec<E>& r, bool whole, int n) {
    if (whole) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < E; i += 4) { const f32x4_any t = {r.v[i], r.v[i + 1], r.v[i + 2], r.v[i + 3]}; if (NT) __builtin_nontemporal_store(t, (f32x4_any*)(p + i)); else *(f32x4_any*)(p + i) = t; }
        } else if constexpr (E == 8) {
            const u32x4_any t = {pack_bf16(r.v[0], r.v[1]), pack_bf16(r.v[2], r.v[3]), pack_bf16(r.v[4], r.v[5]), pack_bf16(r.v[6], r.v[7])};
            if (NT) __builtin_nontemporal_store(t, (u32x4_any*)p); else *(u32x4_any*)p = t;
        } else {
            const u32x2_any t = {pack_bf16(r.v[0], r.v[1]), pack_bf16(r.v[2], r.v[3])};
            if (NT) __builtin_nontemporal_store(t, (u32x2_any*)p); else *(u32x2_any*)p = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < n) p[i] = (T)r.v[i];
    }
}

// where a lane's piece c .. c + E - 1 of a row begins: the piece in which the row ends is moved back to be whole, and what it shares with the piece before is
// worked out twice, to the same values
template <int E>
__device__ __forceinline__ int piece_at(int c, int dim) { return c + E > dim && dim >= E ? dim - E : c; }

__device__ __forceinline__ int64_t load_id(const void* ids, int wide, int64_t i) {
    return wide ? ((const int64_t*)ids)[i] : (int64_t)((const int*)ids)[i];
}

// lpr lanes (a power of two) share a row, each takes every lpr-th piece of E elements; 64 / lpr rows to a wave
template <typename TW, typename TO, int E, bool NT>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* __restrict__ ids, int wide, const TW* __restrict__ w, const float* __restrict__ pos, TO* __restrict__ out,
                                                        int64_t n, int length, int64_t rows, int dim, float scale, int lpr_log2) {
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t r = (wave << (6 - lpr_log2)) + (lane >> lpr_log2);
    if (r >= n) return;
    const int64_t id = load_id(ids, wide, r);
    const bool known = id >= 0 && id < rows;
    const TW* wr = w + (known ? id : 0) * dim;
    const float* pr = pos ? pos + (r % length) * (int64_t)dim : nullptr;
    TO* o = out + r * dim;
    const bool whole = dim >= E;
    for (int first = (lane & ((1 << lpr_log2) - 1)) * E; first < dim; first += E << lpr_log2) {
        const int c = piece_at<E>(first, dim);
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
        store_e<E, TO, NT>(o + c, v, whole, dim - c);
    }
}

// ---- the sort: least significant digit first, stable, two launches for each digit --------------------------------------------------------
#define SORT_THREADS 1024
#define SORT_BLOCKS 256                              // at most: a block's share of the list grows with it

struct SortPass { int shift, bits; };
struct SortPlan { int blocks, passes; int64_t per_block; SortPass pass[4]; };

static SortPlan sort_plan(int64_t n, int64_t rows) {
    SortPlan p;
    int64_t blocks = (n + SORT_THREADS - 1) / SORT_THREADS;
    if (blocks > SORT_BLOCKS) blocks = SORT_BLOCKS;
    p.blocks = (int)(blocks < 1 ? 1 : blocks);
    p.per_block = ((n + p.blocks - 1) / p.blocks + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS;
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

// A fresh gradient's zeros ride along: the sort keeps few CUs busy and waits for latencies, so that each of its launches carries, in the workgroups
// behind its own, an equal part of the fill (152 MB for 49 408 x 768: 20 us at the card's 6.9 TB/s of a fill alone, spread over four launches here).
struct ZeroPart { float* p; int64_t begin, end; int wide, nt; };

__device__ __forceinline__ void zero_part(const ZeroPart& z, int block, int blocks) {
    const int64_t first = z.begin + ((int64_t)block * SORT_THREADS + threadIdx.x) * (z.wide ? 4 : 1);
    const int64_t stride = (int64_t)blocks * SORT_THREADS * (z.wide ? 4 : 1);
    if (z.wide) {                                    // begin, end: multiples of 4
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        if (z.nt) for (int64_t i = first; i < z.end; i += stride) __builtin_nontemporal_store(zero, (f32x4*)(z.p + i));
        else for (int64_t i = first; i < z.end; i += stride) *(f32x4*)(z.p + i) = zero;
    } else {
        for (int64_t i = first; i < z.end; i += stride) z.p[i] = 0.f;
    }
}

// counts of one digit in a block's share; the first pass also turns ids into keys (no row: `rows`, which sorts behind all others)
__global__ __launch_bounds__(SORT_THREADS) void sort_count_kernel(const void* __restrict__ ids, int wide, int64_t rows, int64_t skip, u32* __restrict__ keys, u32* __restrict__ hist, int n,
                                                                  int64_t per_block, int shift, int bits, int sort_blocks, ZeroPart z) {
    if ((int)blockIdx.x >= sort_blocks) { zero_part(z, blockIdx.x - sort_blocks, gridDim.x - sort_blocks); return; }
    __shared__ u32 count[256];
    if (threadIdx.x < 256) count[threadIdx.x] = 0;
    __syncthreads();
    const int64_t b0 = blockIdx.x * per_block;
    const int64_t b1 = b0 + per_block < n ? b0 + per_block : n;
    for (int64_t i = b0 + threadIdx.x; i < b1; i += SORT_THREADS) {
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
    if (threadIdx.x < 256) hist[(int64_t)blockIdx.x * 256 + threadIdx.x] = count[threadIdx.x];
}

// places a block's share behind the smaller digits and behind the earlier blocks' equal ones; `from`: NULL on the first pass (position i)
__global__ __launch_bounds__(SORT_THREADS) void sort_place_kernel(const u32* __restrict__ keys, const u32* __restrict__ from, const u32* __restrict__ hist, u32* __restrict__ keys_out,
                                                                  u32* __restrict__ from_out, int n, int64_t per_block, int shift, int bits, int sort_blocks, ZeroPart z) {
    if ((int)blockIdx.x >= sort_blocks) { zero_part(z, blockIdx.x - sort_blocks, gridDim.x - sort_blocks); return; }
    __shared__ u32 base[256], wcount[16][256], sums[4][2][256], part[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    {   // digit tid & 255: its count in all blocks and in the earlier ones; four threads take every fourth block, eight loads in flight
        const int d = tid & 255, q = tid >> 8;
        u32 before = 0, total = 0;
        for (int b = q; b < sort_blocks; b += 32) {
            u32 h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = b + 4 * i < sort_blocks ? hist[(int64_t)(b + 4 * i) * 256 + d] : 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                total += h[i];
                if (b + 4 * i < (int)blockIdx.x) before += h[i];
            }
        }
        sums[q][0][d] = total;
        sums[q][1][d] = before;
    }
    __syncthreads();
    u32 total = 0, before = 0, incl = 0;
    if (tid < 256) {
#pragma unroll
        for (int q = 0; q < 4; ++q) { total += sums[q][0][tid]; before += sums[q][1][tid]; }
        incl = total;                                // smaller digits: inclusive scan over the wave, then over the four waves
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const u32 t = __shfl_up(incl, o, 64);
            if (lane >= o) incl += t;
        }
        if (lane == 63) part[wave] = incl;
    }
    __syncthreads();
    if (tid < 256) {
        for (int w = 0; w < wave; ++w) incl += part[w];
        base[tid] = incl - total + before;
    }
    const int64_t b0 = blockIdx.x * per_block;
    const int64_t b1 = b0 + per_block < n ? b0 + per_block : n;
    for (int64_t r = b0; r < b1; r += SORT_THREADS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) ((u32*)wcount)[tid + SORT_THREADS * i] = 0;
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
        if (tid < 256) {                             // counts -> places of the waves, in wave order
            u32 at = base[tid];
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                const u32 c = wcount[w][tid];
                wcount[w][tid] = at;
                at += c;
            }
            base[tid] = at;
        }
        __syncthreads();
        if (valid) {
            const u32 at = wcount[wave][digit] + rank;
            keys_out[at] = key;
            from_out[at] = from ? from[i] : (u32)i;
        }
        __syncthreads();
    }
}

// A list that is not long is sorted by counting, in one launch: an entry's place is the number of entries with a smaller key, and of those before it with the same
// key.  A workgroup places TOK entries, a lane each (and 64 / TOK lanes share an entry's comparisons); its 16 waves share the list, which goes through LDS in pieces of
// 4096 keys.  n^2 comparisons, some three instructions for 64 of them.  Whole call with dpos, radix passes -> this:  of 800 rows of 512, 600 tokens 29.2 -> 19.2 us, 4000
// 29.6 -> 19.8, 8000 36.8 -> 28.7, but 12 320 37.7 -> 44.5;  of 49 408 rows of 768 (the zeros are the most of it) 600 tokens 45.1 -> 37.4, 8000 52.4 -> 52.2.
#define RANK_TOKENS 8192
#define RANK_PIECE 4096
template <int TOK>
__global__ __launch_bounds__(SORT_THREADS) void rank_kernel(const void* __restrict__ ids, int wide, int64_t rows, int64_t skip, u32* __restrict__ keys_out, u32* __restrict__ from_out, int n,
                                                            int rank_blocks, ZeroPart z) {
    if ((int)blockIdx.x >= rank_blocks) { zero_part(z, blockIdx.x - rank_blocks, gridDim.x - rank_blocks); return; }
    constexpr int J = 64 / TOK;
    __shared__ u32x4 piece[RANK_PIECE / 4];
    __shared__ u32 count[16 * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int i = blockIdx.x * TOK + lane % TOK, share = lane / TOK;
    const int home = blockIdx.x * TOK & ~63;         // the 64 entries that the workgroup's are among
    const auto key_of = [&](int j) -> u32 {          // (behind the list: larger than any key)
        if (j >= n) return ~0u;
        const int64_t id = load_id(ids, wide, j);
        return id >= 0 && id < rows && id != skip ? (u32)id : (u32)rows;
    };
    const u32 key = key_of(i);
    u32 place = 0;
    for (int j0 = 0; j0 < n; j0 += RANK_PIECE) {
#pragma unroll
        for (int r = 0; r < RANK_PIECE / SORT_THREADS; ++r) ((u32*)piece)[r * SORT_THREADS + tid] = key_of(j0 + r * SORT_THREADS + tid);
        __syncthreads();
#pragma unroll
        for (int b = 0; b < RANK_PIECE / (16 * 64); ++b) {
            const int at = (b * 16 + wave) * 64;     // 64 keys: all before the workgroup's entries, all behind, or the ones that those are among
            if (j0 + at >= n) break;
            if (j0 + at != home) {
                const u32 limit = j0 + at < home ? key + 1 : key;
#pragma unroll
                for (int k = 0; k < 16 / J; ++k) {
                    const u32x4 v = piece[at / 4 + k * J + share];
#pragma unroll
                    for (int e = 0; e < 4; ++e) place += v[e] < limit;
                }
            } else {
                for (int k = 0; k < 16 / J; ++k) {
                    const u32x4 v = piece[at / 4 + k * J + share];
#pragma unroll
                    for (int e = 0; e < 4; ++e) place += v[e] < key || (v[e] == key && j0 + at + (k * J + share) * 4 + e < i);
                }
            }
        }
        __syncthreads();
    }
    count[tid] = place;
    __syncthreads();
    if (tid < TOK && i < n) {
        u32 sum = 0;
#pragma unroll 16
        for (int k = 0; k < 16 * J; ++k) sum += count[k * TOK + tid];
        keys_out[sum] = key;
        from_out[sum] = (u32)i;
    }
}

// ---- the sums over runs of equal keys ----------------------------------------------------------------------------------------------------
enum { RUN_ENDS = 0, RUN_STARTS = 1, RUN_COVERS = 2 };   // nothing; a run that starts in the chunk; one that began before it
struct RunList {
    const u32* keys; const u32* from;                // sorted keys and the positions they came from; keys == NULL: the list of dpos, see run_key
    float* out;                                      // [rows, dim]
    float* part;                                     // [chunks][2][dim]: a chunk's first run where it began earlier, its last where it goes on
    unsigned char* flags;                            // [chunks]: what crosses the border behind the chunk
    int64_t rows;
    int accumulate;
    float scale;
};
struct RunParams {
    RunList list[2];                                 // dweight and dpos, or the one that is wanted
    const void* dy;
    int n, chunk, chunks, dim, length, seqs;         // dpos: entry j is row t = j / seqs of the sequence j % seqs
    int zeros;                                       // this launch zeroes the rows of dweight that no id names (2: past the caches)
};
__device__ __forceinline__ u32 run_key(const RunParams& p, const RunList& l, int j) { return l.keys ? l.keys[j] : (u32)(j / p.seqs); }
__device__ __forceinline__ int64_t run_from(const RunParams& p, const RunList& l, int j) { return l.keys ? (int64_t)l.from[j] : (int64_t)(j % p.seqs) * p.length + j / p.seqs; }

// (own: the first channel of the piece that is not the piece before's too; only those can be added to what is there)
template <int E>
__device__ __forceinline__ void put_row(float* row, int dim, float scale, int accumulate, int c, int own, bool whole, fvec<E> v) {
    float* o = row + c;
#pragma unroll
    for (int i = 0; i < E; ++i) v.v[i] *= scale;
    if (accumulate) {
        if (own > c) {
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (c + i >= own) o[i] += v.v[i];
            return;
        }
        const fvec<E> t = load_e<E, float>(o, whole, dim - c);
#pragma unroll
        for (int i = 0; i < E; ++i) v.v[i] += t.v[i];
    }
    store_e<E, float>(o, v, whole, dim - c);
}

// 16 bytes of dy as they lie in memory (E = 4 of fp32, 8 of bf16): turned into fp32 when they are added, so that eight rows on their way take 32 registers
template <typename T, bool NT>
__device__ __forceinline__ u32x4 raw16(const T* p, bool whole, int n) {
    if (whole) return NT ? __builtin_nontemporal_load((const u32x4_any*)p) : *(const u32x4_any*)p;
    u32x4 r = {0u, 0u, 0u, 0u};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) r[i] = ((const u32*)p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) r[i >> 1] |= (u32)((const unsigned short*)p)[i] << (16 * (i & 1));
    }
    return r;
}
template <typename T, int E>
__device__ __forceinline__ void add_raw16(fvec<E>& acc, const u32x4& r) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc.v[i] += __uint_as_float(r[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { acc.v[2 * i] += bf16_lo_to_f32(r[i]); acc.v[2 * i + 1] += bf16_hi_to_f32(r[i]); }
    }
}

// 16 rows to a wave: each is looked for in the sorted list, and zeroed where it is not
#define ZERO_ROWS 16
__device__ __forceinline__ void zero_unnamed(const RunParams& p) {
    const RunList& l = p.list[0];
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int64_t wave = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * waves + (threadIdx.x >> 6), stride = (int64_t)gridDim.x * gridDim.y * waves * ZERO_ROWS;
    const fvec<4> zero = {{0.f, 0.f, 0.f, 0.f}};
    for (int64_t r0 = wave * ZERO_ROWS; r0 < l.rows; r0 += stride) {
        const int64_t r = r0 + (lane & (ZERO_ROWS - 1));
        int lo = 0, hi = p.n;                        // the first entry whose key is not smaller than r
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if ((int64_t)l.keys[mid] < r) lo = mid + 1; else hi = mid;
        }
        const bool named = lo < p.n && (int64_t)l.keys[lo] == r;
        unsigned todo = (unsigned)__ballot(lane < ZERO_ROWS && r < l.rows && !named);
        while (todo) {
            float* row = l.out + (r0 + __builtin_ctz(todo)) * p.dim;
            todo &= todo - 1;
            for (int own = lane * 4; own < p.dim; own += 256) {
                const int c = piece_at<4>(own, p.dim);
                if (p.zeros > 1) store_e<4, float, true>(row + c, zero, p.dim >= 4, p.dim - c); else store_e<4, float>(row + c, zero, p.dim >= 4, p.dim - c);
            }
        }
    }
}

// blockIdx.x: a chunk of the list blockIdx.z (the last blockIdx.z: zeros, if this launch has them);  eight rows are requested before the first is added (the gather's latency is what there is to hide)
template <typename T, int E, bool NT>
__global__ __launch_bounds__(256) void run_sum_kernel(RunParams p) {
    if (p.zeros && blockIdx.z == gridDim.z - 1) { zero_unnamed(p); return; }
    const RunList& l = p.list[blockIdx.z];
    const int own = (blockIdx.y * 256 + threadIdx.x) * E, c = piece_at<E>(own, p.dim);
    if (own >= p.dim) return;
    const bool whole = p.dim >= E;
    const int j0 = blockIdx.x * p.chunk, j1 = j0 + p.chunk < p.n ? j0 + p.chunk : p.n;
    u32 key = run_key(p, l, j0);
    bool head = j0 > 0 && run_key(p, l, j0 - 1) == key;          // this run began in an earlier chunk
    fvec<E> acc;
#pragma unroll
    for (int i = 0; i < E; ++i) acc.v[i] = 0.f;
    float* part = l.part + (int64_t)blockIdx.x * 2 * p.dim + c;
    if (own == 0) {
        const u32 at_end = run_key(p, l, j1 - 1);
        const bool cross = j1 < p.n && (int64_t)at_end < l.rows && run_key(p, l, j1) == at_end;
        l.flags[blockIdx.x] = (unsigned char)(!cross ? RUN_ENDS : head && key == at_end ? RUN_COVERS : RUN_STARTS);
    }
    for (int j = j0; j < j1 && (int64_t)key < l.rows; j += 8) {
        u32x4 v[8];
        u32 next[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = j + i < j1 ? j + i : j1 - 1;              // (behind the chunk: its last row once more, not added)
            v[i] = raw16<T, NT>((const T*)p.dy + run_from(p, l, at) * p.dim + c, whole, p.dim - c);
            next[i] = at + 1 < p.n ? run_key(p, l, at + 1) : ~0u;   // (~0: no key is that large)
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (j + i < j1 && (int64_t)key < l.rows) {
                add_raw16<T, E>(acc, v[i]);
                if (next[i] != key || j + i + 1 == j1) {
                    if (head) store_e<E, float>(part, acc, whole, p.dim - c);
                    else if (next[i] == key) store_e<E, float>(part + p.dim, acc, whole, p.dim - c);
                    else put_row<E>(l.out + (int64_t)key * p.dim, p.dim, l.scale, l.accumulate, c, own, whole, acc);
#pragma unroll
                    for (int k = 0; k < E; ++k) acc.v[k] = 0.f;
                    head = false;
                    key = next[i];
                }
            }
        }
    }
}

// The runs that cross borders between chunks: for each, its part of the chunk that it starts in and of the chunks behind.  A wave takes a border (and 256
// channels, blockIdx.y): where a run starts in its chunk and goes on into at most JOIN_LIGHT chunks, it adds them by itself, all loads in flight; longer
// runs are left to all 16 waves of the workgroup, which take every 16th chunk each and are added in wave order.
#define JOIN_LIGHT 8
__global__ __launch_bounds__(1024) void run_join_kernel(RunParams p) {
    __shared__ int heavy[16];
    __shared__ float buf[16][256];
    const RunList& l = p.list[blockIdx.z];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int own = (blockIdx.y * 64 + lane) * 4, c = piece_at<4>(own, p.dim);
    const bool mine = own < p.dim, whole = p.dim >= 4;
    const int b = blockIdx.x * 16 + wave;
    int heads = 0;                                               // chunks b + 1 .. b + heads belong to the run that starts in chunk b
    if (b < p.chunks && l.flags[b] == RUN_STARTS) {
        // the chunks behind b that the run covers: the next 64, one to a lane, and for a longer run 1024 at a time, 16 bytes of the list to a lane
        const uint64_t covers = __ballot(b + 1 + lane < p.chunks && l.flags[b + 1 + lane] == RUN_COVERS);
        heads = ~covers ? __builtin_ctzll(~covers) : 64;
        for (int k0 = (b + 65) & ~15, more = covers == ~0ull; more; k0 += 1024) {
            const int k = k0 + lane * 16;
            u32x4 f = {0u, 0u, 0u, 0u};
            if (k < p.chunks) f = *(const u32x4*)(l.flags + k);      // (the list is padded to 16 bytes)
            int n = 0;                                           // this lane's bytes that count (chunks behind b + 64), while the run goes on
            bool on = true;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (k + i > b + 64) {
                    on = on && k + i < p.chunks && ((f[i >> 2] >> (8 * (i & 3))) & 0xffu) == RUN_COVERS;
                    n += on;
                }
            const uint64_t stop = __ballot(!on);
            const int last = stop ? __builtin_ctzll(stop) : 63;
            const int first = k0 <= b + 64 ? 16 - (b + 65 - k0) : 16;      // bytes of lane 0 that count
            heads += last == 0 ? __shfl(n, 0, 64) : first + 16 * (last - 1) + __shfl(n, last, 64);
            more = stop == 0;
        }
        ++heads;                                                 // and the chunk in which it ends
    }
    if (lane == 0) heavy[wave] = heads > JOIN_LIGHT ? heads : 0;
    if (heads > 0 && heads <= JOIN_LIGHT && mine) {
        const float* rest = l.part + ((int64_t)b + 1) * 2 * p.dim + c;
        fvec<4> acc = load_e<4, float>(rest - p.dim, whole, p.dim - c);
        fvec<4> v[JOIN_LIGHT];
#pragma unroll
        for (int u = 0; u < JOIN_LIGHT; ++u)
            if (u < heads) v[u] = load_e<4, float>(rest + (int64_t)u * 2 * p.dim, whole, p.dim - c);
#pragma unroll
        for (int u = 0; u < JOIN_LIGHT; ++u)
            if (u < heads)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc.v[e] += v[u].v[e];
        put_row<4>(l.out + (int64_t)run_key(p, l, (b + 1) * p.chunk) * p.dim, p.dim, l.scale, l.accumulate, c, own, whole, acc);
    }
    __syncthreads();
    for (int i = 0; i < 16; ++i) {
        const int n = heavy[i];
        if (n == 0) continue;                                    // (the same for the whole workgroup)
        const int from = blockIdx.x * 16 + i;
        const float* rest = l.part + ((int64_t)from + 1) * 2 * p.dim + c;
        fvec<4> acc = {{0.f, 0.f, 0.f, 0.f}};
        if (mine) {
            if (wave == 0) acc = load_e<4, float>(rest - p.dim, whole, p.dim - c);
            for (int k = wave; k < n; k += 128) {
                fvec<4> v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = load_e<4, float>(rest + (int64_t)(k + 16 * u < n ? k + 16 * u : k) * 2 * p.dim, whole, p.dim - c);
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (k + 16 * u < n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc.v[e] += v[u].v[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) buf[wave][lane * 4 + e] = acc.v[e];
        __syncthreads();
        if (wave == 0 && mine) {
            for (int q = 1; q < 16; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc.v[e] += buf[q][lane * 4 + e];
            put_row<4>(l.out + (int64_t)run_key(p, l, (from + 1) * p.chunk) * p.dim, p.dim, l.scale, l.accumulate, c, own, whole, acc);
        }
        __syncthreads();
    }
}

__global__ __launch_bounds__(SORT_THREADS) void zero_kernel(ZeroPart z) { zero_part(z, blockIdx.x, gridDim.x); }

// Rows of a chunk: as many workgroups as fit the chip at once (run_sum_kernel leaves room for 7 waves on each of 1024 SIMDs; a second round of them waits for the
// first: 64 x 2048 x 1024 bf16 in chunks of 32 rows 166 us, 40 rows 142, 64 rows 162), whole batches of eight rows, and 16 rows at least, because every
// border between chunks may leave two partial rows (160 x 77 x 768 fp32: 8 rows 68 us, 16 rows 61, 32 rows 65).
#define RUN_WAVES 6600
static int run_waves(int dim, int e) { return (dim + 64 * e - 1) / (64 * e); }
static int run_chunk(int64_t n, int waves) {
    const int64_t c = (n * waves + RUN_WAVES - 1) / RUN_WAVES;
    return (int)(c < 16 ? 16 : (c + 7) / 8 * 8);
}
static int64_t run_chunks(int64_t n, int waves) { return n ? (n + run_chunk(n, waves) - 1) / run_chunk(n, waves) : 0; }

// ---- few tokens: one launch, no sort -----------------------------------------------------------------------------------------------------
// Up to DIRECT_TOKENS tokens (DIRECT_NARROW of rows that one workgroup spans) every workgroup can look at all ids itself.  Three kinds of workgroups, by blockIdx.x:
//   [0, n) if dweight is wanted: a token; the first one of its id finds the others (in ascending order) and sums their rows, the rest of them end
//   then [0, length) if dpos is wanted: a position's rows
//   then the zeros of the rows of dweight that no id names, a range of at most DIRECT_ROWS rows each.
// A workgroup takes 128 pieces of 16 bytes of a row (blockIdx.y); the rows of a sum are dealt out to its 8 (at most 16) sets of threads, whose sums are added in
// order.  All launches with dpos, sorted -> direct:  6 tokens x 512 fp32 9.4 -> 3.7 us, 64 x 768 bf16 18.9 -> 3.9, 512 x 768 fp32 18.4 -> 8.3 (all of one id
// 18.0 -> 12.4);  1001 x 512 fp32 16.6 -> 7.9 (half of one id 17.7 -> 15.8, all of it 15.3 -> 19.5);  wider rows: 1014 x 1024 fp32 19.2 -> 13.2, but of one id
// 19.3 -> 22.6, and 1000 x 2048 bf16 18.9 -> 22.0.
#define DIRECT_TOKENS 512
#define DIRECT_NARROW 1024
#define DIRECT_ROWS 32768
#define DIRECT_PIECES 128
struct DirectParams {
    const void* ids; int wide;
    int64_t rows, skip;
    const void* dy;
    float* dweight; float* dpos;
    int accumulate, n, dim, length, seqs;
    int tokens;                                      // workgroups of tokens: n, or 0 without dweight
    float scale;
    int64_t zero_rows;                               // rows of a zeros' workgroup
};
__device__ __forceinline__ int64_t direct_id(const DirectParams& p, int i) {         // -1: no row
    const int64_t id = load_id(p.ids, p.wide, i);
    return id >= 0 && id < p.rows && id != p.skip ? id : -1;
}
// rows list[0 .. m - 1] of dy, or first, first + step, .. without a list
template <typename T, int E>
__device__ __forceinline__ void direct_sum(const DirectParams& p, const u32* list, int first, int step, int m, float* row, float scale, int accumulate, float (&join)[1024 * E]) {
    const int tid = threadIdx.x, pieces = (p.dim + E - 1) / E, across = pieces < DIRECT_PIECES ? pieces : DIRECT_PIECES;
    const int sets = 1024 / across < 16 ? 1024 / across : 16, set = tid / across, mine = tid % across;
    const int own = (blockIdx.y * DIRECT_PIECES + mine) * E, c = piece_at<E>(own, p.dim);
    const bool whole = p.dim >= E, on = set < sets && own < p.dim;
    fvec<E> acc;
#pragma unroll
    for (int i = 0; i < E; ++i) acc.v[i] = 0.f;
    if (on)
        for (int k = set; k < m; k += 8 * sets) {
            u32x4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = k + i * sets < m ? k + i * sets : k;
                v[i] = raw16<T, false>((const T*)p.dy + (int64_t)(list ? (int)list[j] : first + j * step) * p.dim + c, whole, p.dim - c);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i * sets < m) add_raw16<T, E>(acc, v[i]);
        }
#pragma unroll
    for (int i = 0; i < E; ++i) join[i * 1024 + tid] = acc.v[i];
    __syncthreads();
    if (set > 0 || !on) return;
    for (int q = 1; q < sets && q < m; ++q)
#pragma unroll
        for (int i = 0; i < E; ++i) acc.v[i] += join[i * 1024 + q * across + mine];
    put_row<E>(row, p.dim, scale, accumulate, c, own, whole, acc);
}
template <typename T, int E>
__global__ __launch_bounds__(1024) void direct_kernel(DirectParams p) {
    __shared__ u32 list[DIRECT_ROWS / 32];
    __shared__ int count[16];
    __shared__ float join[1024 * E];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int block = blockIdx.x;
    if (block < p.tokens) {
        const int64_t id = direct_id(p, block);
        if (id < 0) return;
        const bool match = tid < p.n && direct_id(p, tid) == id;
        const uint64_t same = __ballot(match);
        if (lane == 0) count[wave] = __popcll(same);
        __syncthreads();
        int before = 0, m = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) { before += w < wave ? count[w] : 0; m += count[w]; }
        if (match) list[before + __popcll(same & ((1ull << lane) - 1))] = (u32)tid;
        __syncthreads();
        if ((int)list[0] != block) return;
        direct_sum<T, E>(p, list, 0, 0, m, p.dweight + id * p.dim, p.scale, p.accumulate, join);
        return;
    }
    block -= p.tokens;
    if (p.dpos != nullptr) {
        if (block < p.length) {
            direct_sum<T, E>(p, nullptr, block, p.length, p.seqs, p.dpos + (int64_t)block * p.dim, 1.f, 0, join);
            return;
        }
        block -= p.length;
    }
    if (blockIdx.y > 0) return;
    const int64_t r0 = block * p.zero_rows, r1 = r0 + p.zero_rows < p.rows ? r0 + p.zero_rows : p.rows;
    list[tid] = 0;                                   // a bit for each row: named
    __syncthreads();
    if (tid < p.n) {
        const int64_t id = direct_id(p, tid);
        if (id >= r0 && id < r1) atomicOr(&list[(id - r0) >> 5], 1u << ((id - r0) & 31));
    }
    __syncthreads();
    const fvec<4> zero = {{0.f, 0.f, 0.f, 0.f}};
    const unsigned pieces = (unsigned)(p.dim + 3) / 4, all = r1 > r0 ? (unsigned)(r1 - r0) * pieces : 0;
    for (unsigned i = tid; i < all; i += 1024) {
        const unsigned r = i / pieces;
        if ((list[r >> 5] >> (r & 31)) & 1) continue;
        const int c = piece_at<4>((int)(i % pieces) * 4, p.dim);
        store_e<4, float>(p.dweight + (r0 + r) * p.dim + c, zero, p.dim >= 4, p.dim - c);
    }
}

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
#define EFL(TW, TO, E, NT)                                                                                                                       \
    hipLaunchKernelGGL((embed_fwd_kernel<TW, TO, E, NT>), dim3((unsigned)blocks), dim3(256), 0, s, ids, id_bytes == 8, (const TW*)weight, pos, (TO*)out, n, length, rows, dim, scale, l)
#define EF(TW, TO, E)                                                                                                                            \
    do {                                                                                                                                         \
        int l = 0;                                                                                                                               \
        while (l < 6 && ((int64_t)E << l) < dim) ++l;                                                                                            \
        const int64_t waves = (n + (64 >> l) - 1) / (64 >> l), blocks = (waves + 3) / 4;                                                         \
        HH_REQUIRE(hh_grid_fits(blocks, 256), HH_ERR_SHAPE, "hh_embed_tokens_fwd: too many tokens for a launch (%lld of dim %d)", (long long)n, dim); \
        if (n * dim * (int64_t)sizeof(TO) > HH_STREAM_BYTES) EFL(TW, TO, E, true); else EFL(TW, TO, E, false);                                    \
    } while (0)
    if (w_dtype == HH_F32 && out_dtype == HH_F32) EF(float, float, 4);
    else if (w_dtype == HH_F32) EF(float, bf16_t, 4);
    else if (out_dtype == HH_F32) EF(bf16_t, float, 4);
    else EF(bf16_t, bf16_t, 8);
#undef EF
#undef EFL
    return hh_check_launch("hh_embed_tokens_fwd");
}

// (1024 zeros' workgroups at most)
static bool direct_fits(int64_t n, int64_t rows, int dim, int e) { return n <= (dim <= DIRECT_PIECES * e ? DIRECT_NARROW : DIRECT_TOKENS) && rows <= 1024ll * DIRECT_ROWS; }

static int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

extern "C" int64_t hh_workspace_bytes_embed_tokens_bwd(int64_t seqs, int length, int64_t rows, int dim) {
    if (!embed_shape_ok(seqs, length, rows, dim)) return -1;
    const int64_t n = seqs * length;
    if (direct_fits(n, rows, dim, 4)) return 0;
    const int64_t chunks = run_chunks(n, run_waves(dim, 8));                         // (bf16; fp32 rows take more waves, and fewer chunks)
    return 4 * align256(4 * n) + align256(SORT_BLOCKS * 256 * 4) + 2 * align256(chunks) + 2 * align256(chunks * 2 * (int64_t)dim * 4);
}

// part i of `parts` of the zeros of out, and the workgroups that write it.  Large gradients are zeroed past the caches: 160 x 77 of 49 408 x 768 fp32 with a few outputs in
// turn 67.5 -> 58.3 us (59.4 -> 57.9 with one output's memory over and over), 64 x 2048 of 49 408 x 1024 bf16 147.4 -> 141.5 (137.5 -> 140.7).
static ZeroPart zero_share(float* out, int64_t total, int i, int parts, int* blocks) {
    ZeroPart z = {out, 0, 0, 0, total * 4 > HH_STREAM_BYTES};
    *blocks = 0;
    if (out == nullptr) return z;
    z.wide = HH_ALIGNED16(out) && total % 4 == 0;
    const int64_t share = ((total + parts - 1) / parts + 3) / 4 * 4;
    z.begin = i * share < total ? i * share : total;
    z.end = z.begin + share < total ? z.begin + share : total;
    const int64_t want = (z.end - z.begin + 16383) / 16384;                   // 16 values for each thread
    *blocks = (int)(want < 1024 ? want : 1024);
    return z;
}

extern "C" int hh_embed_tokens_bwd(const void* ids, int id_bytes, const void* dy, int dy_dtype, float* dweight, int accumulate, float* dpos, int64_t seqs, int length, int64_t rows,
                                   int dim, float scale, int64_t skip_id, void* workspace, hh_stream_t stream) {
    HH_REQUIRE(embed_shape_ok(seqs, length, rows, dim), HH_ERR_SHAPE, "hh_embed_tokens_bwd: need length, rows, dim > 0, dim <= 2^20 and fewer than 2^30 tokens and 2^31 rows (seqs=%lld length=%d rows=%lld dim=%d)",
               (long long)seqs, length, (long long)rows, dim);
    HH_REQUIRE(id_bytes == 4 || id_bytes == 8, HH_ERR_DTYPE, "hh_embed_tokens_bwd: ids are 4 or 8 bytes wide");
    HH_REQUIRE(dy_dtype == HH_F32 || dy_dtype == HH_BF16, HH_ERR_DTYPE, "hh_embed_tokens_bwd: bad dtype");
    HH_REQUIRE(dweight != nullptr || dpos != nullptr, HH_ERR_ALIGN, "hh_embed_tokens_bwd: dweight and dpos are NULL");
    hipStream_t s = (hipStream_t)stream;
    const int64_t n = seqs * length;
    const int e = dy_dtype == HH_F32 ? 4 : 8;
    const bool direct = direct_fits(n, rows, dim, e);
    HH_REQUIRE(n == 0 || ((ids != nullptr || dweight == nullptr) && dy != nullptr && (direct || (workspace != nullptr && HH_ALIGNED16(workspace)))), HH_ERR_ALIGN,
               "hh_embed_tokens_bwd: ids, dy and a 16-byte aligned workspace are needed");
    int zb = 0;
    float* zero = accumulate ? nullptr : dweight;
    // zeros beside the sort, for all of dweight, or beside the sums, for the rows that no id names: where there are as many tokens as rows most rows are named, and are
    // not written twice (131 072 tokens of 49 408 x 1024, spread evenly 153 -> 136 us, by Zipf's law 144 -> 138, all of one id 144 -> 153; 50 000 of 49 408 x 768
    // 90.5 -> 81.6, 87 -> 84, 97 -> 105; 12 320 of 10 000 x 768 no difference)
    const bool late = zero != nullptr && n > RANK_TOKENS && n >= rows;
    if (n == 0) {
        ZeroPart z = zero_share(zero, rows * dim, 0, 1, &zb);
        if (zb) hipLaunchKernelGGL(zero_kernel, dim3(zb), dim3(SORT_THREADS), 0, s, z);
        z = zero_share(dpos, (int64_t)length * dim, 0, 1, &zb);
        if (zb) hipLaunchKernelGGL(zero_kernel, dim3(zb), dim3(SORT_THREADS), 0, s, z);
        return hh_check_launch("hh_embed_tokens_bwd");
    }
    if (direct) {
        int64_t zeros = zero == nullptr ? 0 : (rows * dim + 16383) / 16384;
        zeros = zeros > 1024 ? 1024 : zeros;
        const int64_t least = zero == nullptr ? 0 : (rows + DIRECT_ROWS - 1) / DIRECT_ROWS;
        if (zeros < least) zeros = least;
        DirectParams p = {ids, id_bytes == 8, rows, skip_id, dy, dweight, dpos, accumulate != 0, (int)n, dim, length, (int)seqs, dweight ? (int)n : 0, scale, zeros ? (rows + zeros - 1) / zeros : 0};
        const int across = e * DIRECT_PIECES;
        const dim3 grid((unsigned)(p.tokens + (dpos ? length : 0) + zeros), (unsigned)((dim + across - 1) / across));
        if (dy_dtype == HH_F32) hipLaunchKernelGGL((direct_kernel<float, 4>), grid, dim3(1024), 0, s, p);
        else hipLaunchKernelGGL((direct_kernel<bf16_t, 8>), grid, dim3(1024), 0, s, p);
        return hh_check_launch("hh_embed_tokens_bwd");
    }
    char* ws = (char*)workspace;
    u32* keys[2] = {(u32*)ws, (u32*)(ws + align256(4 * n))};
    u32* from[2] = {(u32*)(ws + 2 * align256(4 * n)), (u32*)(ws + 3 * align256(4 * n))};
    u32* hist = (u32*)(ws + 4 * align256(4 * n));
    unsigned char* flags = (unsigned char*)hist + align256(SORT_BLOCKS * 256 * 4);
    const int64_t chunks = run_chunks(n, run_waves(dim, e)), flag_bytes = align256(chunks), part_bytes = align256(chunks * 2 * (int64_t)dim * 4);
    char* part = (char*)flags + 2 * flag_bytes;
    const SortPlan sp = sort_plan(n, rows);
    int sorted = sp.passes & 1;                                                   // the buffers that hold the sorted list
    if (dweight != nullptr && n <= RANK_TOKENS) {                                 // (dpos has its list without a sort)
        const int tok = n <= 4096 ? 16 : 32, blocks = (int)((n + tok - 1) / tok);          // about a workgroup to a CU
        const ZeroPart z = zero_share(zero, rows * dim, 0, 1, &zb);
#define RANK(T) hipLaunchKernelGGL((rank_kernel<T>), dim3(blocks + zb), dim3(SORT_THREADS), 0, s, ids, id_bytes == 8, rows, skip_id, keys[0], from[0], (int)n, blocks, z)
        if (tok == 16) RANK(16); else RANK(32);
#undef RANK
        sorted = 0;
    } else if (dweight != nullptr) {
        for (int i = 0; i < sp.passes; ++i) {
            ZeroPart z = zero_share(late ? nullptr : zero, rows * dim, 2 * i, 2 * sp.passes, &zb);
            hipLaunchKernelGGL(sort_count_kernel, dim3(sp.blocks + zb), dim3(SORT_THREADS), 0, s, i == 0 ? ids : nullptr, id_bytes == 8, rows, skip_id, keys[i & 1], hist, (int)n, sp.per_block,
                               sp.pass[i].shift, sp.pass[i].bits, sp.blocks, z);
            z = zero_share(late ? nullptr : zero, rows * dim, 2 * i + 1, 2 * sp.passes, &zb);
            hipLaunchKernelGGL(sort_place_kernel, dim3(sp.blocks + zb), dim3(SORT_THREADS), 0, s, keys[i & 1], i == 0 ? nullptr : from[i & 1], hist, keys[(i + 1) & 1], from[(i + 1) & 1], (int)n,
                               sp.per_block, sp.pass[i].shift, sp.pass[i].bits, sp.blocks, z);
        }
    }
    RunParams p;
    p.dy = dy; p.n = (int)n; p.chunk = run_chunk(n, run_waves(dim, e)); p.chunks = (int)chunks; p.dim = dim; p.length = length; p.seqs = (int)seqs;
    p.zeros = !late ? 0 : rows * dim * 4 > HH_STREAM_BYTES ? 2 : 1;
    p.list[0] = RunList{keys[sorted], from[sorted], dweight, (float*)part, flags, rows, accumulate != 0, scale};
    p.list[1] = RunList{nullptr, nullptr, dpos, (float*)(part + part_bytes), flags + flag_bytes, length, 0, 1.f};
    const int need = (dim + e - 1) / e;
    const int threads = need >= 256 ? 256 : (need + 63) / 64 * 64;
    const unsigned lists = (dweight ? 1u : 0u) + (dpos ? 1u : 0u);
    if (dweight == nullptr) p.list[0] = p.list[1];
    const dim3 grid((unsigned)p.chunks, (unsigned)((need + 255) / 256), lists + (late ? 1u : 0u));
    // dy past the caches where it is read once (64 x 2048 x 1024 bf16: 150 -> 142 us) or does not fit there; with both gradients it is read twice, and 160 x 77 x 768 fp32
    // stay in the cache between (58.5 us, 64.7 past it)
    const bool nt = lists == 1 || n * dim * (e == 4 ? 4 : 2) > HH_STREAM_BYTES;
    if (e == 4 && nt) hipLaunchKernelGGL((run_sum_kernel<float, 4, true>), grid, dim3(threads), 0, s, p);
    else if (e == 4) hipLaunchKernelGGL((run_sum_kernel<float, 4, false>), grid, dim3(threads), 0, s, p);
    else if (nt) hipLaunchKernelGGL((run_sum_kernel<bf16_t, 8, true>), grid, dim3(threads), 0, s, p);
    else hipLaunchKernelGGL((run_sum_kernel<bf16_t, 8, false>), grid, dim3(threads), 0, s, p);
    if (p.chunks > 1)
        hipLaunchKernelGGL(run_join_kernel, dim3((unsigned)((p.chunks + 15) / 16), (unsigned)((dim + 255) / 256), lists), dim3(1024), 0, s, p);
    return hh_check_launch("hh_embed_tokens_bwd");
}
