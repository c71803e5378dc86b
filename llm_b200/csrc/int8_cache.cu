// A step's keys and values appended to a paged cache held in 8 bits (int8_pages.cuh), the rotation by the position on the way.
//
//   queries[t, a] = R(p_t) q[t, a]            keys of token t: R(p_t) k[t, h], values: v[t, h], rounded to whole numbers of their block's scale
//   R: (x0, x1) -> (x0 c - x1 s, x1 c + x0 s) for each pair of the first n_rot elements, c and s from a 32-bit table of angles by position
//
// A warp does one row of queries, or all new rows of one block of one head's keys or values: the largest magnitude, the scale, then the whole
// numbers. A block that is continued keeps its scale where that is enough; where it grows, the rows in front of the new ones are divided by the growth
// and rounded again. Which of a step's tokens begins a block's rows (the first of the block, or of its sequence) does the block's work, so no two
// warps write to one block and nothing depends on the order of blocks.
//
// All arithmetic is in 32 bits with a rounding for each product and sum (no contraction), so that a row's whole numbers do not depend on how
// the compiler joins them.
#include "int8_pages.cuh"
#include "tc.cuh"

using namespace llmb;

LLMB_DEFINE_LAST_ERROR(llmb_int8_cache)

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

struct Args {
    const void* qkv;                 // [n_tokens, (n_heads + 2 n_kv_heads) * dim]
    const float* angles;             // [positions, n_rot]: cosines, then sines; or none
    const int* tok_pos;
    const int* tok_seq;
    const int* cu_seqlens;
    const int* block_table;
    void* queries;                   // [n_tokens, n_heads * dim]
    signed char* keys;
    float* key_scales;
    signed char* values;
    float* value_scales;
    int table_stride, ring_pages, n_heads, n_kv_heads, dim, n_rot, interleaved, write_cache;
    int block;                       // positions of a block
    int n_tokens, n_seqs, n_pages, n_positions;
};

// What the kernel reports of a place outside of what the call was given: a position without angles, a sequence or a page that there is not, a token
// that is not its sequence's, a sequence that brings more than its ring holds. Nothing is read or written there.
constexpr int OUT_OF_RANGE = 51;

// Whether the rows begin .. end - 1 of a sequence, of which `token` has `position`, go to pages of their own: with more of them than the ring has, two
// warps would write to one block.
__device__ __forceinline__ bool fits_ring(const Args& a, int token, int position, int begin, int end) {
    const int first = max(position - (token - begin), 0), last = position + (end - 1 - token);
    return last / LLMB_PAGE - first / LLMB_PAGE < a.ring_pages;
}

// the two elements of pair p: rotated pairs first, then neighbours of the part that is not
__device__ __forceinline__ void pair_at(const Args& a, int p, bool turned, int& i0, int& i1) {
    const int half = a.n_rot >> 1;
    if (turned && p < half && !a.interleaved) {
        i0 = p;
        i1 = p + half;
    } else {
        i0 = 2 * p;
        i1 = 2 * p + 1;
    }
}
template <typename T>
__device__ __forceinline__ void load_pair(const Args& a, const T* row, const float* angles, int p, bool turned, int i0, int i1, float& x0, float& x1) {
    x0 = to_float(row[i0]);
    x1 = to_float(row[i1]);
    const int half = a.n_rot >> 1;
    if (turned && p < half) {
        const float c = angles[p], s = angles[half + p], low = x0;
        x0 = __fsub_rn(__fmul_rn(low, c), __fmul_rn(x1, s));
        x1 = __fadd_rn(__fmul_rn(x1, c), __fmul_rn(low, s));
    }
}
__device__ __forceinline__ signed char whole(float x, float inverse) { return (signed char)__float2int_rn(__fmul_rn(x, inverse)); }

template <typename T>
__global__ void __launch_bounds__(THREADS) int8_append_kernel(const __grid_constant__ Args a, int* status) {
    griddep_launch();
    griddep_wait();
    const int lane = threadIdx.x & 31, unit = blockIdx.y * WARPS + (threadIdx.x >> 5), token = blockIdx.x;
    const int D = a.dim, pairs = D >> 1, units = a.n_heads + 2 * a.n_kv_heads;
    if (unit >= units) return;
    const T* qkv = behind_wait(static_cast<const T*>(a.qkv));
    const size_t row_stride = (size_t)units * D;
    if (token >= a.cu_seqlens[a.n_seqs]) return;              // a row behind the last sequence's
    const int position = a.tok_pos[token];
    const bool turned = unit < a.n_heads + a.n_kv_heads;      // queries and keys
    auto angles_of = [&](int pos) { return a.angles + (size_t)pos * a.n_rot; };
    if (position < 0 || (a.angles && position >= a.n_positions)) {
        if (lane == 0 && status) atomicCAS(status, 0, OUT_OF_RANGE);
        return;
    }
    if (unit < a.n_heads) {
        const T* from = qkv + token * row_stride + (size_t)unit * D;
        T* to = static_cast<T*>(a.queries) + ((size_t)token * a.n_heads + unit) * D;
        for (int p = lane; p < pairs; p += 32) {
            int i0, i1;
            float x0, x1;
            pair_at(a, p, true, i0, i1);
            load_pair(a, from, angles_of(position), p, true, i0, i1, x0, x1);
            to[i0] = from_float<T>(x0);
            to[i1] = from_float<T>(x1);
        }
        return;
    }
    if (!a.write_cache) return;
    const int seq = a.tok_seq[token], first = position % a.block;
    int page = -1, n_rows = 0;
    if ((unsigned)seq < (unsigned)a.n_seqs) {
        const int begin = a.cu_seqlens[seq], end = a.cu_seqlens[seq + 1];
        if (token >= begin && token < end) {
            if (first != 0 && token != begin) return;         // another warp has this block
            n_rows = min(a.block - first, end - token);
            if (fits_ring(a, token, position, begin, end)) page = a.block_table[(size_t)seq * a.table_stride + (position / LLMB_PAGE) % a.ring_pages];
        }
    }
    if ((unsigned)page >= (unsigned)a.n_pages || token + n_rows > a.n_tokens || (a.angles && position + n_rows > a.n_positions)) {
        if (lane == 0 && status) atomicCAS(status, 0, OUT_OF_RANGE);
        return;
    }
    const int head = turned ? unit - a.n_heads : unit - a.n_heads - a.n_kv_heads;
    const int row = position % LLMB_PAGE, per = LLMB_PAGE / a.block;
    const size_t at = (size_t)page * a.n_kv_heads + head;
    signed char* to = (turned ? a.keys : a.values) + (at * LLMB_PAGE + row) * D;
    float* scale_at = (turned ? a.key_scales : a.value_scales) + at * per + row / a.block;

    const T* from = qkv + token * row_stride + (size_t)unit * D;
    uint32_t most = 0;
    for (int r = 0; r < n_rows; ++r)
        for (int p = lane; p < pairs; p += 32) {
            int i0, i1;
            float x0, x1;
            pair_at(a, p, turned, i0, i1);
            load_pair(a, from + r * row_stride, angles_of(position + r), p, turned, i0, i1, x0, x1);
            most = max(most, max(__float_as_uint(x0) & 0x7fffffffu, __float_as_uint(x1) & 0x7fffffffu));
        }
    float scale = __uint_as_float(scale_bits(__reduce_max_sync(0xffffffffu, most)));
    if (first != 0) {                                         // the block is continued
        const float before = *scale_at;
        __syncwarp();                                         // (everyone has read it)
        if (!is_number(scale) || !is_number(before)) {
            scale = __uint_as_float(0x7fffffffu);
        } else if (scale > before) {
            const float shrink = before / scale;
            signed char* older = to - (size_t)first * D;
            for (int i = lane; i < first * D; i += 32) older[i] = whole((float)older[i], shrink);
        } else {
            scale = before;
        }
    }
    const float inverse = is_number(scale) ? 1.f / scale : 0.f;
    for (int r = 0; r < n_rows; ++r)
        for (int p = lane; p < pairs; p += 32) {
            int i0, i1;
            float x0, x1;
            pair_at(a, p, turned, i0, i1);
            load_pair(a, from + r * row_stride, angles_of(position + r), p, turned, i0, i1, x0, x1);
            to[(size_t)r * D + i0] = inverse != 0.f ? whole(x0, inverse) : 0;
            to[(size_t)r * D + i1] = inverse != 0.f ? whole(x1, inverse) : 0;
        }
    if (lane == 0) *scale_at = scale;
}

// ------------------------------------------------------------------------------------------------ 16 bytes at a time
//
// Heads of 64 and 128 that rotate as a whole or not at all. Eight pairs of elements are a lane's: two pieces of a row, which with the angles it holds
// in registers for all of a token's queries; D / 16 lanes a row, so a warp has 4 rows (8) to an instruction. A block of the cache is one warp's, up to
// 16 new rows of it in registers between the largest magnitude and the whole numbers (more are read twice).
//
// A block of threads does `run` neighbouring tokens: their first rows in blocks of the cache are looked up by one warp, then the eight warps take
// blocks and queries in turn. Rows are
// held as they came and rotated again for the whole numbers: with the rotated values in registers there was room for half as many warps (16,889 tokens 95 us
// for 80). Those tokens (32 heads over 8 of 128) move 389 MB, at 4.9 TB/s: a warp's loads are 4 KB, with 16 to 24 warps on an SM. Three and four blocks of
// 80 and 64 registers spilled (78 and 104 us; 64 tokens 3.9 and 4.9). What a step of 64 tokens takes (3.1 us) is a launch and three dependent reads.

constexpr int MAX_RUN = 16, HELD = 16, QUERIES = 4;            // tokens of a block of threads; rows that a warp holds; rows of queries, in instructions

struct Begun {                                                 // a block of the cache that begins to be written with a token
    int token, position, n_rows, page;
};

// eight values as they are in memory
template <typename T> struct Raw {
    uint4 v[sizeof(T) / 2];
};
template <typename T> __device__ __forceinline__ Raw<T> raw8(const T* p) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
template <typename T> __device__ __forceinline__ void unpack8(const Raw<T>& r, float (&x)[8]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 2) x[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
        else x[i] = __uint_as_float(w[i]);
    }
}
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&x)[8]) { unpack8(raw8(p), x); }
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(p) = make_uint4(tc::pack2(x[0], x[1]), tc::pack2(x[2], x[3]), tc::pack2(x[4], x[5]), tc::pack2(x[6], x[7]));
    } else {
        *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(x);
        *reinterpret_cast<float4*>(p + 4) = *reinterpret_cast<const float4*>(x + 4);
    }
}
__device__ __forceinline__ uint2 whole8(const float (&x)[8], float inverse) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)__float2int_rn(__fmul_rn(x[i], inverse)) & 0xffu) << (8 * (i & 3));
    return make_uint2(w[0], w[1]);
}

// A lane's part of a row: eight pairs. Interleaved, the two pieces adjoin and the pairs lie inside; otherwise they are half a head apart.
template <typename T, int D, bool INTERLEAVED> struct Row {
    static constexpr int LANES = D / 16, ROWS = 32 / LANES;
    static __device__ __forceinline__ int first(int lane) { return (lane % LANES) * (INTERLEAVED ? 16 : 8); }
    static constexpr int APART = INTERLEAVED ? 8 : D / 2;
    static __device__ __forceinline__ void turn(float (&a)[8], float (&b)[8], const float (&c)[8], const float (&s)[8]) {
        auto pair = [&](float& low, float& high, int i) {
            const float x = low;
            low = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(high, s[i]));
            high = __fadd_rn(__fmul_rn(high, c[i]), __fmul_rn(x, s[i]));
        };
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                pair(a[2 * i], a[2 * i + 1], i);
                pair(b[2 * i], b[2 * i + 1], 4 + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) pair(a[i], b[i], i);
        }
    }
};
__device__ __forceinline__ uint32_t largest8(const float (&x)[8]) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
    return most;
}

template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS) int8_append_vec_kernel(const __grid_constant__ Args a, int run, int* status) {
    using R = Row<T, D, INTERLEAVED>;
    constexpr int LANES = R::LANES, ROWS = R::ROWS, STEPS = HELD / ROWS, HALF = D / 2;
    __shared__ Begun begun[MAX_RUN];
    __shared__ int n_begun, positions[MAX_RUN];
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row_in = lane / LANES, first_pair = lane % LANES * 8;
    const int token0 = blockIdx.x * run, n_here = min(run, a.n_tokens - token0), units = a.n_heads + 2 * a.n_kv_heads;
    // (positions, sequences and tables are not written by the kernels of a step)
    if (warp == 0) {
        Begun b{};
        bool mine = false;
        if (lane < n_here) positions[lane] = -1;
        if (lane < n_here && token0 + lane < a.cu_seqlens[a.n_seqs]) {           // (rows behind the last sequence's are left as they are)
            b.token = token0 + lane;
            b.position = a.tok_pos[b.token];
            const int seq = a.tok_seq[b.token];
            bool there = b.position >= 0 && !(a.angles && b.position >= a.n_positions);
            if (there) positions[lane] = b.position;
            if (there && a.write_cache) {
                int begin = 0, end = 0;
                if ((unsigned)seq < (unsigned)a.n_seqs) {
                    begin = a.cu_seqlens[seq];
                    end = a.cu_seqlens[seq + 1];
                }
                there = b.token >= begin && b.token < end;
                if (there && (b.position % a.block == 0 || b.token == begin)) {
                    int place = b.position / LLMB_PAGE;
                    if (place >= a.ring_pages) place %= a.ring_pages;
                    b.n_rows = min(a.block - b.position % a.block, end - b.token);
                    b.page = a.block_table[(size_t)seq * a.table_stride + place];
                    there = mine = (unsigned)b.page < (unsigned)a.n_pages && b.token + b.n_rows <= a.n_tokens &&
                                   !(a.angles && b.position + b.n_rows > a.n_positions) && fits_ring(a, b.token, b.position, begin, end);
                }
            }
            if (!there && status) atomicCAS(status, 0, OUT_OF_RANGE);
        }
        const unsigned which = __ballot_sync(0xffffffffu, mine);
        if (mine) begun[__popc(which & ((1u << lane) - 1u))] = b;
        if (lane == 0) n_begun = __popc(which);
    }
    __syncthreads();
    griddep_wait();
    const T* qkv = behind_wait(static_cast<const T*>(a.qkv));
    const size_t row_stride = (size_t)units * D;
    auto angles_of = [&](int position, float (&c)[8], float (&s)[8]) {
        const float* from = a.angles + (size_t)position * D + first_pair;
        load8(from, c);
        load8(from + HALF, s);
    };
    // ---- blocks of the cache: (begun block, keys or values, head)
    const int n_blocks = n_begun * 2 * a.n_kv_heads, stride = gridDim.y * WARPS;
    int task = blockIdx.y * WARPS + warp;
    for (; task < n_blocks; task += stride) {
        const Begun b = begun[task / (2 * a.n_kv_heads)];
        const int unit = task % (2 * a.n_kv_heads);            // of the projection, behind the queries
        const bool keys = unit < a.n_kv_heads, turned = keys && a.angles;
        const int head = keys ? unit : unit - a.n_kv_heads, first = b.position % a.block, row = b.position % LLMB_PAGE;
        const T* from = qkv + b.token * row_stride + (size_t)(a.n_heads + unit) * D + R::first(lane);
        const size_t at = (size_t)b.page * a.n_kv_heads + head;
        signed char* block_rows = (keys ? a.keys : a.values) + (at * LLMB_PAGE + row) * D;
        signed char* to = block_rows + R::first(lane);
        float* scale_at = (keys ? a.key_scales : a.value_scales) + at * (LLMB_PAGE / a.block) + row / a.block;
        const float before = first != 0 ? *scale_at : 0.f;
        Raw<T> low[STEPS], high[STEPS];                        // as they came: rotated for the magnitude, and again for the whole numbers
        auto fetch = [&](int r0) {                             // rows r0 + i * ROWS + row_in: to place i
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int r = r0 + i * ROWS + row_in;
                if (r < b.n_rows) {
                    low[i] = raw8(from + r * row_stride);
                    high[i] = raw8(from + r * row_stride + R::APART);
                }
            }
        };
        auto values_of = [&](int r, int i, float (&x)[8], float (&y)[8]) {
            unpack8(low[i], x);
            unpack8(high[i], y);
            if (turned) {
                float c[8], s[8];
                angles_of(b.position + r, c, s);
                R::turn(x, y, c, s);
            }
        };
        uint32_t most = 0;
        for (int r0 = 0; r0 < b.n_rows; r0 += HELD) {
            fetch(r0);
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int r = r0 + i * ROWS + row_in;
                if (r < b.n_rows) {
                    float x[8], y[8];
                    values_of(r, i, x, y);
                    most = max(most, max(largest8(x), largest8(y)));
                }
            }
        }
        float scale = __uint_as_float(scale_bits(__reduce_max_sync(0xffffffffu, most)));
        if (first != 0) {                                      // the block is continued
            __syncwarp();                                      // (everyone has read its scale)
            if (!is_number(scale) || !is_number(before)) {
                scale = __uint_as_float(0x7fffffffu);
            } else if (scale > before) {
                const float shrink = before / scale;
                signed char* older = block_rows - first * D;
                for (int i = lane; i < first * D / 16; i += 32) {
                    uint4 v = reinterpret_cast<uint4*>(older)[i];
                    signed char* q = reinterpret_cast<signed char*>(&v);
#pragma unroll
                    for (int k = 0; k < 16; ++k) q[k] = whole((float)q[k], shrink);
                    reinterpret_cast<uint4*>(older)[i] = v;
                }
            } else {
                scale = before;
            }
        }
        const float inverse = is_number(scale) ? 1.f / scale : 0.f;
        for (int r0 = 0; r0 < b.n_rows; r0 += HELD) {
            if (b.n_rows > HELD) fetch(r0);
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int r = r0 + i * ROWS + row_in;
                if (r < b.n_rows) {
                    float x[8], y[8];
                    values_of(r, i, x, y);
                    *reinterpret_cast<uint2*>(to + r * D) = inverse != 0.f ? whole8(x, inverse) : make_uint2(0u, 0u);
                    *reinterpret_cast<uint2*>(to + r * D + R::APART) = inverse != 0.f ? whole8(y, inverse) : make_uint2(0u, 0u);
                }
            }
        }
        if (lane == 0) *scale_at = scale;
    }
    // ---- queries: (token, QUERIES times ROWS heads), all of them under way at once
    const int chunks = (a.n_heads + ROWS * QUERIES - 1) / (ROWS * QUERIES), n_chunks = n_here * chunks;
    for (task -= n_blocks; task < n_chunks; task += stride) {
        const int t = task / chunks, head0 = (task - t * chunks) * ROWS * QUERIES + row_in, position = positions[t];
        if (position < 0) continue;
        const T* from = qkv + (token0 + t) * row_stride + R::first(lane);
        T* to = static_cast<T*>(a.queries) + (size_t)(token0 + t) * a.n_heads * D + R::first(lane);
        Raw<T> low[QUERIES], high[QUERIES];
        float c[8], s[8];
        if (a.angles) angles_of(position, c, s);
#pragma unroll
        for (int i = 0; i < QUERIES; ++i)
            if (head0 + i * ROWS < a.n_heads) {
                low[i] = raw8(from + (head0 + i * ROWS) * D);
                high[i] = raw8(from + (head0 + i * ROWS) * D + R::APART);
            }
#pragma unroll
        for (int i = 0; i < QUERIES; ++i)
            if (head0 + i * ROWS < a.n_heads) {
                float x[8], y[8];
                unpack8(low[i], x);
                unpack8(high[i], y);
                if (a.angles) R::turn(x, y, c, s);
                store8(to + (head0 + i * ROWS) * D, x);
                store8(to + (head0 + i * ROWS) * D + R::APART, y);
            }
    }
}

template <typename T, int D>
void launch_vec(const Args& a, int* status, cudaStream_t stream) {
    // blocks of threads for every SM several times, up to MAX_RUN tokens each
    int run = a.n_tokens / (148 * 4);
    run = run < 1 ? 1 : run > MAX_RUN ? MAX_RUN : run;
    // few tokens: a token's work over several blocks of threads
    const int blocks = (a.n_tokens + run - 1) / run, heads = Row<T, D, false>::ROWS * QUERIES;                // of queries, to a task
    const int tasks = (a.write_cache ? 2 * a.n_kv_heads : 0) + (a.n_heads + heads - 1) / heads, most = (tasks + WARPS - 1) / WARPS;
    int slices = 148 * 4 / blocks;
    slices = slices > most ? most : slices < 1 ? 1 : slices;
    const dim3 grid(blocks, slices);
    if (a.interleaved) llmb::launch(int8_append_vec_kernel<T, D, true>, grid, dim3(THREADS), 0, stream, true, a, run, status);
    else llmb::launch(int8_append_vec_kernel<T, D, false>, grid, dim3(THREADS), 0, stream, true, a, run, status);
}

}  // namespace

LLMB_EXPORT int llmb_int8_cache_status() {
    int* s = tc::status_word();
    if (!s) return -1;
    int v = *s;
    *s = 0;
    return v;
}

// The sizes of a call, one integer each.
struct llmb_int8_append_sizes {
    int dtype, table_stride, ring_pages, n_tokens, n_seqs, n_pages;
    int n_heads, n_kv_heads, head_dim, n_rot, n_positions, interleaved, block, write_cache;
};

LLMB_EXPORT int llmb_int8_append(const void* qkv, const float* angles, const int* tok_pos, const int* tok_seq, const int* cu_seqlens,
                                 const int* block_table, void* queries, void* keys, float* key_scales, void* values, float* value_scales,
                                 const llmb_int8_append_sizes* sizes, cudaStream_t stream) {
    const llmb_int8_append_sizes& z = *sizes;
    if (z.n_tokens == 0 || z.n_seqs == 0) return LLMB_OK;
    LLMB_REQUIRE(z.dtype == LLMB_DTYPE_F32 || z.dtype == LLMB_DTYPE_BF16, "int8_append: unknown dtype %d", z.dtype);
    LLMB_REQUIRE(z.n_tokens > 0 && z.n_seqs > 0 && z.n_heads > 0 && z.n_kv_heads > 0 && z.ring_pages > 0, "int8_append: bad sizes");
    LLMB_REQUIRE(z.head_dim > 0 && z.head_dim % 2 == 0 && z.head_dim <= LLMB_MAX_HEAD_DIM, "int8_append: head_dim %d must be even and at most %d", z.head_dim,
                 LLMB_MAX_HEAD_DIM);
    LLMB_REQUIRE(z.n_rot >= 0 && z.n_rot <= z.head_dim && z.n_rot % 2 == 0, "int8_append: the rotated part %d must be even and at most head_dim %d", z.n_rot,
                 z.head_dim);
    LLMB_REQUIRE(z.block >= 1 && z.block <= LLMB_PAGE && (z.block & (z.block - 1)) == 0, "int8_append: blocks of %d positions", z.block);
    const bool turns = angles != nullptr && z.n_rot > 0;
    Args a{qkv, turns ? angles : nullptr, tok_pos, tok_seq, cu_seqlens, block_table, queries, (signed char*)keys, key_scales, (signed char*)values,
           value_scales, z.table_stride, z.ring_pages, z.n_heads, z.n_kv_heads, z.head_dim, turns ? z.n_rot : 0, z.interleaved, z.write_cache, z.block,
           z.n_tokens, z.n_seqs, z.n_pages, z.n_positions};
    const int units = z.n_heads + (z.write_cache ? 2 * z.n_kv_heads : 0);
    const int rows = ceil_div(units, WARPS);
    LLMB_REQUIRE(rows <= 65535, "int8_append: too many heads");
    static int* status = nullptr;                // (one address for all devices)
    if (!status && tc::status_word()) LLMB_CUDA(cudaHostGetDevicePointer((void**)&status, tc::status_word(), 0));
    auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    if ((z.head_dim == 64 || z.head_dim == 128) && (a.n_rot == 0 || a.n_rot == z.head_dim) && aligned(qkv) && aligned(queries) && aligned(keys) &&
        aligned(values) && aligned(angles)) {
        if (z.dtype == LLMB_DTYPE_F32) z.head_dim == 64 ? launch_vec<float, 64>(a, status, stream) : launch_vec<float, 128>(a, status, stream);
        else z.head_dim == 64 ? launch_vec<__nv_bfloat16, 64>(a, status, stream) : launch_vec<__nv_bfloat16, 128>(a, status, stream);
        return check_launch("int8_append_vec");
    }
    dim3 grid(z.n_tokens, rows);
    if (z.dtype == LLMB_DTYPE_F32) llmb::launch(int8_append_kernel<float>, grid, dim3(THREADS), 0, stream, true, a, status);
    else llmb::launch(int8_append_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, stream, true, a, status);
    return check_launch("int8_append");
}

LLMB_PACKED(llmb_int8_append)
