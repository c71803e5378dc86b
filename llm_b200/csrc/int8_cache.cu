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

// What the kernel reports of a place outside of what the call was given: a position without angles, a sequence or a page that there is not. Nothing is
// read or written there.
constexpr int OUT_OF_RANGE = 51;

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
        if (first != 0 && token != a.cu_seqlens[seq]) return; // another warp has this block
        n_rows = min(a.block - first, a.cu_seqlens[seq + 1] - token);
        page = a.block_table[(size_t)seq * a.table_stride + (position / LLMB_PAGE) % a.ring_pages];
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
    if (z.n_tokens == 0) return LLMB_OK;
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
    int* status = nullptr;
    if (tc::status_word()) LLMB_CUDA(cudaHostGetDevicePointer((void**)&status, tc::status_word(), 0));
    dim3 grid(z.n_tokens, rows);
    if (z.dtype == LLMB_DTYPE_F32) llmb::launch(int8_append_kernel<float>, grid, dim3(THREADS), 0, stream, true, a, status);
    else llmb::launch(int8_append_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, stream, true, a, status);
    return check_launch("int8_append");
}

LLMB_PACKED(llmb_int8_append)
