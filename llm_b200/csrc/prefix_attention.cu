// Attention of a batch whose sequences share their first pages of the cache: several samples of one prompt, several questions
// behind one document. Sequences that stand together in the batch form groups; the members of a group have the same pages in the
// first `group_pages` places of their page tables. The keys and values of those pages are read once for all queries of the group, or by
// each sequence where they are few pages (plan_for).
//
//   out[t, a] = sum_j p_j v_j,  p = softmax_j(scale * q[t, a] . k_j),  j <= position of t,  keys of head a * kv_heads / heads
//
// The sum over j is cut into parts: slices of the shared pages, where the rows of a tile are the queries of all members, and slices
// of each sequence's own pages, where they are its own queries. Each part leaves, per row, (weighted values, maximum, sum); the last
// kernel joins them with out = sum_i acc_i e^(m_i - m) / sum_i l_i e^(m_i - m) in the order of the parts.
//
// A row of a tile is (token, query head of the key head): row r of a range of tokens is token r / share, head r % share, with
// share = heads / kv_heads, so that one pass over a key head serves all query heads that share it.
//
// Everything that changes from step to step (lengths, tables, groups) is read from device arrays; the sizes of the launch are upper
// bounds (most tokens of a group, most pages) and a block beyond the real work leaves; a step of more tokens than its bounds say is
// reported. A key beyond a row's position has no weight whatever is stored there, and values beyond the last position of a sequence's own pages are
// taken for zero, so that what an earlier sequence left in a page (infinities and NaN too) does not reach a result. Shared pages are full: every
// member of the group holds all their positions, and nothing in them is left over. A row that sees no key is zero.
#include "mma.cuh"
#include "prefix_plan.h"
#include "tc.cuh"

using namespace llmb;
using namespace llmb::tc;
using namespace llmb_prefix;

LLMB_DEFINE_LAST_ERROR(llmb_prefix_attention)

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_SLOTS = 2 * MAX_SPLITS;         // of a row: parts of the shared pages, of own ones

struct Args {
    const void* q;
    const void* k_cache;
    const void* v_cache;
    const int* block_table;          // [n_seqs, table_stride]
    const int* seq_lens;             // [n_seqs] with the new tokens
    const int* cu_seqlens;           // [n_seqs + 1]
    const int* group_first;          // [n_groups + 1] the first sequence of each group
    const int* group_pages;          // [n_groups] pages that the group's members share
    void* out;
    float* acc;                      // [rows, slots, head_dim], a row a (token, head), or a row of the tiles that are cut (`whole`)
    float* stats;                    // [rows, slots, 2]: maximum in base-2 units, sum
    int q_stride, out_stride, table_stride, n_seqs, n_groups, n_heads, n_kv_heads, head_dim;
    float scale_log2;
    int prefix_tiles, prefix_splits, own_tiles, own_splits, slots;
    int vectors;                     // the caches' rows can be read 16 bytes at a time
    int full_tiles;                  // tiles of the wide kernel whose walk is one block's; the others are cut into prefix_splits pieces
    int even_blocks;                 // > 0: so many blocks share the groups' pages in slices of equal length, else every group is cut into prefix_splits
    int behind;                      // own parts launched behind the wide kernel, which has waited for all that they read
    int longest_first;               // own slices in the order of their sequences' own pages (prefix_attention_few_kernel)
    const int* order;                // that order, in the block's shared memory, or none
    int alone;                       // every sequence reads its shared pages for itself: own parts start at the first page
    int whole;                       // a tile of a group walks its sequences' own pages behind the shared ones (tensor cores)
};

// A block's share of the work: rows of a range of tokens against a slice of pages.
struct Item {
    int kv_head, tile, tiles, slot;
    int seq_first, seq_last;         // the sequences whose tokens are the rows
    int first_token, n_rows;
    int page_first;                  // the first page that is not shared (own parts)
    int page_begin, page_end;        // of the table of seq_first
};

__device__ __forceinline__ int group_of(const Args& a, int seq) {
    int low = 0, high = a.n_groups - 1;                       // the last group whose first sequence is not behind seq
    while (low < high) {
        int mid = (low + high + 1) >> 1;
        if (a.group_first[mid] <= seq) low = mid;
        else high = mid - 1;
    }
    return low;
}

// x: the block's number; false where nothing is left for it
__device__ __forceinline__ bool item_of(const Args& a, int x, Item& w) {
    w.kv_head = x % a.n_kv_heads;
    x /= a.n_kv_heads;
    int prefix_blocks = a.even_blocks ? 0 : a.n_groups * a.prefix_tiles * a.prefix_splits;
    int share = a.n_heads / a.n_kv_heads;
    if (x < prefix_blocks) {
        w.tiles = a.prefix_tiles;
        w.tile = x % w.tiles;
        x /= w.tiles;
        int split = x % a.prefix_splits, group = x / a.prefix_splits;
        w.seq_first = a.group_first[group];
        w.seq_last = a.group_first[group + 1];
        int pages = a.group_pages[group], per = (pages + a.prefix_splits - 1) / a.prefix_splits;
        w.page_first = 0;
        w.page_begin = min(split * per, pages);
        w.page_end = min(w.page_begin + per, pages);
        w.slot = split;
    } else {
        x -= prefix_blocks;
        w.tiles = a.own_tiles;
        w.tile = x % w.tiles;
        x /= w.tiles;
        int split = x % a.own_splits, seq = x / a.own_splits;
        if (a.order) seq = a.order[seq];
        w.seq_first = seq;
        w.seq_last = seq + 1;
        int first = a.alone ? 0 : a.group_pages[group_of(a, seq)], last = (a.seq_lens[seq] + LLMB_PAGE - 1) / LLMB_PAGE;
        int pages = max(last - first, 0), per = (pages + a.own_splits - 1) / a.own_splits;
        w.page_first = first;
        w.page_begin = first + min(split * per, pages);
        w.page_end = first + min(split * per + per, pages);
        w.slot = a.prefix_splits + split;
    }
    if (w.seq_first >= w.seq_last) return false;
    w.first_token = a.cu_seqlens[w.seq_first];
    w.n_rows = (a.cu_seqlens[w.seq_last] - w.first_token) * share;
    return true;
}

// which of the item's sequences a token belongs to, and its position there
__device__ __forceinline__ int sequence_of(const Args& a, const Item& w, int token) {
    int low = w.seq_first, high = w.seq_last - 1;             // the last sequence whose tokens do not start behind this one
    while (low < high) {
        int mid = (low + high + 1) >> 1;
        if (a.cu_seqlens[mid] <= token) low = mid;
        else high = mid - 1;
    }
    return low;
}
__device__ __forceinline__ int position_of(const Args& a, const Item& w, int token) {
    int seq = sequence_of(a, w, token);
    return a.seq_lens[seq] - a.cu_seqlens[seq + 1] + token;
}

// The arrays that say which sequences there are, in shared memory (one round of loads) where there is room.
constexpr int STAGED_SEQS = 512;
struct Staged {
    int seq_lens[STAGED_SEQS], cu_seqlens[STAGED_SEQS + 1], group_first[STAGED_SEQS + 1], group_pages[STAGED_SEQS];
};
__device__ __forceinline__ void stage_arrays(Args& a, Staged& s) {
    if (a.n_seqs > STAGED_SEQS) return;
    for (int i = threadIdx.x; i <= a.n_seqs; i += blockDim.x) {
        s.cu_seqlens[i] = a.cu_seqlens[i];
        if (i < a.n_seqs) s.seq_lens[i] = a.seq_lens[i];
        if (i <= a.n_groups) s.group_first[i] = a.group_first[i];
        if (i < a.n_groups) s.group_pages[i] = a.group_pages[i];
    }
    __syncthreads();
    a.seq_lens = s.seq_lens;
    a.cu_seqlens = s.cu_seqlens;
    a.group_first = s.group_first;
    a.group_pages = s.group_pages;
}

// ------------------------------------------------------------------------------------------------ any type, any head size
//
// 32-bit arithmetic on the CUDA cores: the path of 32-bit caches, and of the head sizes that the tensor-core kernel is not built for.
// A block holds 32 rows and walks its pages one by one: 64 keys and values in shared memory (as 32-bit values), four rows a warp. A lane
// forms their scores with keys `lane` and `lane + 32`, shares maxima and sums with the others, and adds the weighted values of its columns, two
// multiply-adds to an instruction. Rows of a key or value are 4 words longer than the head, so that the eight rows that are read at a time lie in
// different banks. 32-bit pages come by cp.async, the values during the scores and the next keys during the products with the values.
//
// Eight sequences behind 4,096 positions (32 heads of 64, 32-bit): 24.9 us; the products alone are 4. What bounds it is a page's chain: with two blocks on an SM
// the scores take 4,300 cycles, the softmax 1,300, the values 3,000, where reading shared memory alone is 1,500 a block and scores or values (every
// warp reads the page again for four rows). With two rows and four keys to a thread of half a warp it was 27, loads through registers row by row 36,
// single multiply-adds 25.7, three blocks an SM of 80 registers a thread 33.

constexpr int SIMT_ROWS = 32, SIMT_THREADS = 256, RT = SIMT_ROWS / (SIMT_THREADS / 32);     // RT: rows of a warp

// two 32-bit values to an instruction
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) { return pair_of(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float half_of(uint64_t v, int which) { return __uint_as_float((uint32_t)(which ? v >> 32 : v)); }
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(x), "l"(y), "l"(z));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
    return v;
}

template <int DMAX>
constexpr int simt_floats() { return (SIMT_ROWS + 2 * LLMB_PAGE) * (DMAX + 4) + SIMT_ROWS * LLMB_PAGE + SIMT_ROWS + 4; }

template <typename T, int DMAX>
__global__ void __launch_bounds__(SIMT_THREADS) prefix_attention_simt_kernel(const __grid_constant__ Args args) {
    constexpr int LD = DMAX + 4, W = DMAX == 64 ? 2 : 4, COLS = DMAX / (32 * W);      // a lane's columns: COLS times W that adjoin
    extern __shared__ __align__(16) float smem[];
    float* qs = smem;                              // [32][LD], scaled
    float* ks = qs + SIMT_ROWS * LD;               // [64][LD]
    float* vs = ks + LLMB_PAGE * LD;               // [64][LD]
    float* ps = vs + LLMB_PAGE * LD;               // [warp][64 keys][4 rows]
    int* row_pos = reinterpret_cast<int*>(ps + SIMT_ROWS * LLMB_PAGE);
    int* last_pos = row_pos + SIMT_ROWS;
    __shared__ Staged staged;

    griddep_launch();
    Args a = args;
    stage_arrays(a, staged);
    Item w;
    const bool work = item_of(a, blockIdx.x, w);
    griddep_wait();
    if (!work) return;
    const int tid = threadIdx.x, ty = tid >> 5, tx = tid & 31;
    const int D = a.head_dim, share = a.n_heads / a.n_kv_heads;
    const T* q = static_cast<const T*>(a.q);
    const T* k_cache = static_cast<const T*>(a.k_cache);
    const T* v_cache = static_cast<const T*>(a.v_cache);
    const int* pages = a.block_table + (size_t)w.seq_first * a.table_stride;

    constexpr int V = 16 / sizeof(T);
    const int width = a.vectors ? D / V : (D + 3) & ~3;        // of a row, in vectors or in single values (the scores read four at a time)
    const int row_step = SIMT_THREADS / width, first_row = tid / width, col = (tid - first_row * width) * (a.vectors ? V : 1);
    // a page's keys or values: thread tid takes column `col` of every row_step-th row (rows wider than the block: all columns in turn)
    auto load = [&](float* to, const T* cache, int page) {
        const T* from = cache + ((size_t)page * a.n_kv_heads + w.kv_head) * LLMB_PAGE * D;
        if (!a.vectors) {
            for (int i = tid; i < LLMB_PAGE * width; i += SIMT_THREADS) {
                int row = i / width, c = i - row * width;
                to[row * LD + c] = c < D ? to_float(from[(size_t)row * D + c]) : 0.f;
            }
        } else if (first_row < row_step) {
#pragma unroll 4
            for (int row = first_row; row < LLMB_PAGE; row += row_step) {
                if constexpr (sizeof(T) == 4) {
                    cp_async16(to + row * LD + col, from + (size_t)row * D + col);
                } else {
                    __align__(16) T x[V];
                    *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(from + (size_t)row * D + col);
#pragma unroll
                    for (int j = 0; j < V; j += 4)
                        *reinterpret_cast<float4*>(to + row * LD + col + j) = make_float4(to_float(x[j]), to_float(x[j + 1]), to_float(x[j + 2]), to_float(x[j + 3]));
                }
            }
        }
        cp_async_commit();
    };

    for (int tile = w.tile; tile * SIMT_ROWS < w.n_rows; tile += w.tiles) {
        int row0 = tile * SIMT_ROWS, rows = min(SIMT_ROWS, w.n_rows - row0);
        __syncthreads();                           // the tile before is done with shared memory
#pragma unroll 4
        for (int r = tid >> 5; r < SIMT_ROWS; r += SIMT_THREADS / 32) {          // a warp a row
            const bool valid = r < rows;
            const int token = w.first_token + (row0 + (valid ? r : 0)) / share, head = w.kv_head * share + (row0 + (valid ? r : 0)) % share;
            const T* from = q + (size_t)token * a.q_stride + (size_t)head * D;
#pragma unroll
            for (int d = tid & 31; d < DMAX; d += 32) qs[r * LD + d] = valid && d < D ? to_float(from[d]) * a.scale_log2 : 0.f;
        }
        if (tid < SIMT_ROWS) {
            int p = tid < rows ? position_of(a, w, w.first_token + (row0 + tid) / share) : -1;
            row_pos[tid] = p;
            p = __reduce_max_sync(0xffffffffu, p);
            if (tid == 0) *last_pos = p;
        }
        __syncthreads();
        const int last = *last_pos;                // the last position that a row of the tile sees
        const int end = min(w.page_end, last < 0 ? 0 : last / LLMB_PAGE + 1);

        float m[RT], l[RT];
        uint64_t o[RT / 2][COLS * W];                  // of rows 2 i and 2 i + 1
        float4* weights = reinterpret_cast<float4*>(ps) + ty * LLMB_PAGE;
        int pos[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
            pos[i] = row_pos[ty * RT + i];
        }
#pragma unroll
        for (int i = 0; i < RT / 2; ++i)
#pragma unroll
            for (int c = 0; c < COLS * W; ++c) o[i][c] = 0;
        const bool idle = ty * RT >= rows;                     // a warp without rows
        int page = w.page_begin < end ? pages[w.page_begin] : 0;
        if (w.page_begin < end) load(ks, k_cache, page);
        for (int logical = w.page_begin; logical < end; ++logical) {
            const int key0 = logical * LLMB_PAGE, stored = min(LLMB_PAGE, last + 1 - key0);
            cp_async_wait<0>();
            __syncthreads();                       // the keys are there, everyone is done with the values before
            load(vs, v_cache, page);
            if (logical + 1 < end) page = pages[logical + 1];
            if (!idle) {
                uint64_t dot[RT][2];                   // even and odd columns apart
#pragma unroll
                for (int i = 0; i < RT; ++i) dot[i][0] = dot[i][1] = 0;
#pragma unroll 4
                for (int d = 0; d < D; d += 4) {
                    ulonglong2 qv[RT], kv[2];
#pragma unroll
                    for (int i = 0; i < RT; ++i) qv[i] = *reinterpret_cast<const ulonglong2*>(qs + (ty * RT + i) * LD + d);
#pragma unroll
                    for (int j = 0; j < 2; ++j) kv[j] = *reinterpret_cast<const ulonglong2*>(ks + (tx + 32 * j) * LD + d);
#pragma unroll
                    for (int i = 0; i < RT; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j) dot[i][j] = fma2(qv[i].x, kv[j].x, fma2(qv[i].y, kv[j].y, dot[i][j]));
                }
                float weight[2][RT], alpha[RT];
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    float s[2], top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        s[j] = key0 + tx + 32 * j > pos[i] ? -INFINITY : half_of(dot[i][j], 0) + half_of(dot[i][j], 1);
                        top = fmaxf(top, s[j]);
                    }
                    top = warp_max(top);
                    float new_m = fmaxf(m[i], top), against = new_m == -INFINITY ? 0.f : new_m;
                    alpha[i] = exp2f(m[i] - against);
                    m[i] = new_m;
                    float add = 0.f;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        weight[j][i] = exp2f(s[j] - against);
                        add += weight[j][i];
                    }
                    l[i] = l[i] * alpha[i] + add;      // of this thread's keys
                }
                static_assert(RT == 4, "a key's weights of a warp's rows are one load");
#pragma unroll
                for (int j = 0; j < 2; ++j) weights[tx + 32 * j] = make_float4(weight[j][0], weight[j][1], weight[j][2], weight[j][3]);
#pragma unroll
                for (int i = 0; i < RT / 2; ++i)
#pragma unroll
                    for (int c = 0; c < COLS * W; ++c) o[i][c] = fma2(o[i][c], pair_of(alpha[2 * i], alpha[2 * i + 1]), 0);
            }
            cp_async_wait<0>();
            __syncthreads();                       // the values are there, everyone is done with the keys
            if (logical + 1 < end) load(ks, k_cache, page);
            if (stored < LLMB_PAGE) {              // values behind the last position are whatever the page held: zero here
                for (int row = stored + ty; row < LLMB_PAGE; row += SIMT_THREADS / 32)
                    for (int d = tx; d < D; d += 32) vs[row * LD + d] = 0.f;
                __syncthreads();
            }
            if (idle) continue;
#pragma unroll 8
            for (int j = 0; j < LLMB_PAGE; ++j) {
                const ulonglong2 p = *reinterpret_cast<const ulonglong2*>(weights + j);
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    if (c * 32 * W >= D) break;               // (lanes behind the head's last column add what no one reads)
                    float v[W];
                    const float* from = vs + j * LD + (c * 32 + tx) * W;
                    if constexpr (W == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(from);
                    else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(from);
#pragma unroll
                    for (int x = 0; x < W; ++x) {
                        const uint64_t twice = pair_of(v[x], v[x]);
                        o[0][c * W + x] = fma2(p.x, twice, o[0][c * W + x]);
                        o[1][c * W + x] = fma2(p.y, twice, o[1][c * W + x]);
                    }
                }
            }
            __syncwarp();                     // the weights are read before the next page's are written
        }
        if (!idle) {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                l[i] = warp_sum(l[i]);
                int r = ty * RT + i;
                if (r >= rows) continue;
                int token = w.first_token + (row0 + r) / share, head = w.kv_head * share + (row0 + r) % share;
                if (a.slots == 1) {
                    float inv = l[i] > 0.f ? 1.f / l[i] : l[i] == 0.f ? 0.f : l[i];      // (a NaN stays one)
                    T* to = static_cast<T*>(a.out) + (size_t)token * a.out_stride + (size_t)head * D;
#pragma unroll
                    for (int c = 0; c < COLS; ++c)
#pragma unroll
                        for (int x = 0; x < W; ++x)
                            if ((c * 32 + tx) * W + x < D) to[(c * 32 + tx) * W + x] = from_float<T>(half_of(o[i / 2][c * W + x], i & 1) * inv);
                } else {
                    size_t slot = ((size_t)token * a.n_heads + head) * a.slots + w.slot;
#pragma unroll
                    for (int c = 0; c < COLS; ++c)
#pragma unroll
                        for (int x = 0; x < W; ++x)
                            if ((c * 32 + tx) * W + x < D) a.acc[slot * D + (c * 32 + tx) * W + x] = half_of(o[i / 2][c * W + x], i & 1);
                    if (tx == 0) {
                        a.stats[slot * 2] = m[i];
                        a.stats[slot * 2 + 1] = l[i];
                    }
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ bfloat16, up to 128 rows
//
// What a decode step brings: a group's shared pages against up to 128 rows, a sequence's own pages against up to 16. Reading the pages is the
// work; two blocks an SM hold a slice of pages each.
//
// Items of 16 rows or fewer (prefix_attention_few_kernel): warp 4 keeps a ring of pages in flight (TMA, 64 x 64 boxes with the 128-byte
// swizzle); warps 0 to 3 take 16 of a page's 64 keys each with mma.sync.m16n8k16 and keep a maximum, a sum and weighted values of their own, in
// 32 bits, which are merged at the end. mma.sync stands up to that many rows: with 64 rows a page took four times as long as on tcgen05.
//
// Items of more rows (prefix_attention_tile_kernel): S[128, 64 keys] = Q K^T into one of two buffers of scores in tensor memory (warp 1), the
// weights written over them by a thread a row (warps 2 to 5; those without rows only pass the word on), O[128, D] += P V with P from tensor
// memory. The scores of the page after the next are issued behind P V of this one.
//
// In both, weights are rounded to 8 bits, what the tensor cores take, and their sum is of the unrounded ones. The two are kernels of their own:
// as branches of one, the own pages of a step took a third longer.

constexpr int TC_ROWS = TILE_ROWS;                // lanes of tensor memory
constexpr int KV_PIECE = LLMB_PAGE * 64 * 2;      // a page, 64 columns of the head: 8 KB
constexpr int Q_PIECE = TC_ROWS * 64 * 2;         // 128 rows, 64 columns of the head: 16 KB
constexpr int FEW_THREADS = 160, TILE_THREADS = 192;
constexpr int FEW_WARPS = 4;
// tensor memory of an item: two buffers of scores (64 columns of 32-bit values, the weights over the first 32), O beside them
constexpr uint32_t S_COL = 0, O_COL = 128, TMEM_COLS = 256;

// where element (row, col) of a page lies in shared memory: pieces of 64 columns, 16-byte chunks swizzled by the row
__device__ __forceinline__ const unsigned char* swizzled(const unsigned char* page, int row, int col) {
    return page + (col >> 6) * KV_PIECE + row * 128 + ((((col >> 3) & 7) ^ (row & 7)) << 4);
}

// Sequences by their own pages, most first: where there are more blocks than fit at once, long slices that start last would leave most SMs idle. A
// thread a sequence counts those in front of it.
constexpr int ORDERED_SEQS = 128;
struct Order {
    int4 keys[ORDERED_SEQS / 4];
    int at[ORDERED_SEQS];
};
__device__ __forceinline__ void order_sequences(Args& a, Order& order) {
    if (!a.longest_first) return;
    const int i = threadIdx.x, n = (a.n_seqs + 3) / 4;
    int mine = -1, rank = 0;
    if (i < a.n_seqs) {
        const int pages = (a.seq_lens[i] + LLMB_PAGE - 1) / LLMB_PAGE - (a.alone ? 0 : a.group_pages[group_of(a, i)]);
        mine = (max(pages, 0) << 8) + ORDERED_SEQS - i;      // (no two are alike)
    }
    if (i < 4 * n) reinterpret_cast<int*>(order.keys)[i] = mine;
    __syncthreads();
    if (i < a.n_seqs) {
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
            const int4 k = order.keys[j];
            rank += (k.x > mine) + (k.y > mine) + (k.z > mine) + (k.w > mine);
        }
        order.at[rank] = i;
    }
    __syncthreads();
    a.order = order.at;
}

template <int HD> struct Ring {
    static constexpr int STAGE = 2 * (HD / 64) * KV_PIECE;   // a page's keys and values
    static constexpr int STAGES = HD == 64 ? 6 : 3;          // two blocks an SM: 192 KB in flight
    static constexpr int MERGE = FEW_WARPS * 16 * (HD + 8 + 2) * 4;
    static constexpr int BYTES = STAGE * STAGES;
    static_assert(MERGE <= BYTES, "the merge takes the ring's place");
    static_assert((HD / 64) * (Q_PIECE + 4 * KV_PIECE) <= BYTES, "the queries and two pages");
};

// Slices of equal length of groups of unequal ones: `per` pages each, the least number (two at least) with which all groups' slices fit into the
// blocks that there are for a key head, or a group's all. Each warp finds out for itself, a lane a group. w: the slice's group and pages; *pieces:
// the slices of the group; false where nothing is left for the block.
__device__ __forceinline__ bool even_slice_of(const Args& a, int x, int lane, Item& w, int& pieces) {
    const unsigned all = 0xffffffffu;
    const int share = a.n_heads / a.n_kv_heads, heads = a.even_blocks / a.n_kv_heads;          // blocks of a key head
    auto pages_of = [&](int g) { return g < a.n_groups && a.cu_seqlens[a.group_first[g + 1]] > a.cu_seqlens[a.group_first[g]] ? a.group_pages[g] : 0; };
    int work = 0, items = 0, most = 0;
    for (int g0 = 0; g0 < a.n_groups; g0 += 32) {
        int pages = pages_of(g0 + lane);
        work += __reduce_add_sync(all, pages);
        items += __popc(__ballot_sync(all, pages > 0));
        most = max(most, __reduce_max_sync(all, pages));
    }
    int per = items < heads ? (work + heads - items - 1) / (heads - items) : most;
    per = max(max(per, 2), (most + a.prefix_splits - 1) / a.prefix_splits);
    w.kv_head = x % a.n_kv_heads;
    x /= a.n_kv_heads;
    for (int g0 = 0; g0 < a.n_groups; g0 += 32) {
        int pages = pages_of(g0 + lane), mine = (pages + per - 1) / per, before = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            int left = __shfl_up_sync(all, before, d);
            if (lane >= d) before += left;
        }
        unsigned beyond = __ballot_sync(all, x < before);
        if (!beyond) {
            x -= __shfl_sync(all, before, 31);
            continue;
        }
        int at = __ffs(beyond) - 1;
        pieces = __shfl_sync(all, mine, at);
        x -= __shfl_sync(all, before - mine, at);
        pages = __shfl_sync(all, pages, at);
        w.seq_first = a.group_first[g0 + at];
        w.seq_last = a.group_first[g0 + at + 1];
        w.page_first = 0;
        w.page_begin = min(x * per, pages);
        w.page_end = min(x * per + per, pages);
        w.slot = x;
        w.tile = 0;
        w.tiles = 1;
        w.first_token = a.cu_seqlens[w.seq_first];
        w.n_rows = (a.cu_seqlens[w.seq_last] - w.first_token) * share;
        return true;
    }
    return false;
}

// A part's maximum and sum. Where slices are of equal length, the last one of a group leaves the parts that it has fewer than there is room for, and
// the own part of a sequence that shares nothing those of the shared pages.
__device__ __forceinline__ void put_stats(const Args& a, const Item& w, int pieces, size_t row, float m, float sum) {
    float2* stats = reinterpret_cast<float2*>(a.stats) + row * a.slots;
    stats[w.slot] = make_float2(sum != 0.f ? m : -INFINITY, sum);
    if (!a.even_blocks) return;
    int first = a.prefix_splits;
    if (w.slot == a.prefix_splits && w.page_first == 0) first = 0;
    else if (w.slot == pieces - 1) first = pieces;
    for (int i = first; i < a.prefix_splits; ++i) stats[i] = make_float2(-INFINITY, 0.f);
}

// What a kernel reports of a step that brings more tokens than the bounds of its call say (no wait has this code).
constexpr int BEYOND_BOUNDS = 50;
__device__ __forceinline__ void report_beyond_bounds(int* status) {
    if (threadIdx.x == 0 && status) atomicCAS(status, 0, BEYOND_BOUNDS);
}

// The block's slice; uniform for the block. *pieces: of a group whose slices are dealt out. The kernels have room for `most` rows, which the launch has
// chosen them for by max_new and max_group; the lengths are on the device only, so that it shows here whether they keep to those.
__device__ __forceinline__ bool slice_of(const Args& a, Item& w, int& pieces, int most, int* status) {
    int x = blockIdx.x - (a.prefix_tiles > 0 ? a.even_blocks : 0);
    pieces = 0;
    bool work = (x < 0 ? even_slice_of(a, blockIdx.x, threadIdx.x & 31, w, pieces) : item_of(a, x, w)) && w.n_rows > 0;
    if (work && w.n_rows > most) {
        report_beyond_bounds(status);
        w.n_rows = most;
    }
    return work;
}

// Up to 16 rows over the pages [page_begin, page_end) of one table.
template <int HD>
__global__ void __launch_bounds__(FEW_THREADS, 2)
prefix_attention_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                            const __grid_constant__ Args args, int* status) {
    constexpr int STAGES = Ring<HD>::STAGES, STAGE = Ring<HD>::STAGE, PIECES = HD / 64;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(base + Ring<HD>::BYTES);
    uint64_t* empty = full + STAGES;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + STAGES);
    __shared__ Staged staged;

    griddep_launch();
    const int warp = warp_index(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(smem_u32(&full[i]), 1);
            mbar_init(smem_u32(&empty[i]), FEW_WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    Args a = args;
    stage_arrays(a, staged);                                 // (lengths, groups and tables are not written by the kernels of a step)
    __shared__ Order order;
    order_sequences(a, order);
    Item w;
    int pieces;
    const bool work = slice_of(a, w, pieces, FEW_ROWS, status);
    __syncthreads();
    // Behind the kernel of the shared parts the own ones may run beside them: that kernel lets them start when the one in front of it is
    // complete. Each block waits for it at its end, so that the join waits for both.
    if (!a.behind || !work) griddep_wait();
    if (!work) return;
    const int share = a.n_heads / a.n_kv_heads;
    const bool own = w.slot >= a.prefix_splits;
    const int last_token = w.first_token + (w.n_rows - 1) / share;
    int limit = w.page_end * LLMB_PAGE - 1;                  // the last position that a row sees of these pages
    if (own) limit = min(limit, a.seq_lens[w.seq_first] - a.cu_seqlens[w.seq_first + 1] + last_token);
    const int n_pages = min(w.page_end, limit < 0 ? 0 : limit / LLMB_PAGE + 1) - w.page_begin;

    const int g = lane >> 2, t = lane & 3, part = warp;      // warps 0 to 3: 16 keys of every page
    float acc[HD / 8][4], run_max[2] = {-INFINITY, -INFINITY}, run_sum[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
    if (warp == FEW_WARPS) {
        const int* pages = a.block_table + (size_t)w.seq_first * a.table_stride + w.page_begin;
        int numbers = lane < n_pages ? pages[lane] : 0;      // 32 places of the table at once
        for (int i = 0; i < n_pages; ++i) {
            if (i > 0 && (i & 31) == 0) numbers = i + lane < n_pages ? pages[i + lane] : 0;
            int stage = i % STAGES;
            int row = (__shfl_sync(0xffffffffu, numbers, i & 31) * a.n_kv_heads + w.kv_head) * LLMB_PAGE;
            if (i >= STAGES && !mbar_wait_warp(smem_u32(&empty[stage]), (i / STAGES - 1) & 1, abort_flag, status, 21)) break;
            if (elect_one()) {
                uint32_t bar = smem_u32(&full[stage]);
                mbar_expect_tx(bar, STAGE);
                for (int h = 0; h < PIECES; ++h) tma_load_2d(smem_u32(base + stage * STAGE + h * KV_PIECE), &map_k, bar, h * 64, row);
                for (int h = 0; h < PIECES; ++h) tma_load_2d(smem_u32(base + stage * STAGE + (PIECES + h) * KV_PIECE), &map_v, bar, h * 64, row);
            }
            __syncwarp();
        }
    } else {
        // rows g and g + 8 of the mma tile are this lane's
        uint32_t qa[HD / 16][4];
        int pos[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            int r = g + half * 8;
            bool valid = r < w.n_rows;
            int token = w.first_token + (valid ? r : 0) / share, head = w.kv_head * share + (valid ? r : 0) % share;
            pos[half] = valid ? position_of(a, w, token) : -1;
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + (size_t)token * a.q_stride + (size_t)head * HD;
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                qa[ks][half] = valid ? *reinterpret_cast<const uint32_t*>(q + ks * 16 + 2 * t) : 0u;
                qa[ks][2 + half] = valid ? *reinterpret_cast<const uint32_t*>(q + ks * 16 + 8 + 2 * t) : 0u;
            }
        }
        for (int i = 0; i < n_pages; ++i) {
            int stage = i % STAGES;
            if (!mbar_wait_warp(smem_u32(&full[stage]), (i / STAGES) & 1, abort_flag, status, 22)) break;
            const unsigned char* k_page = base + stage * STAGE;
            const unsigned char* v_page = k_page + PIECES * KV_PIECE;
            const int key0 = (w.page_begin + i) * LLMB_PAGE + part * 16;
            if (key0 <= limit) {
                float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    uint32_t b[4];
                    ldmatrix_x4(b, swizzled(k_page, part * 16 + (lane >> 4) * 8 + (lane & 7), ks * 16 + ((lane >> 3) & 1) * 8));
                    mma_bf16(s0, qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b[0], b[1]);
                    mma_bf16(s1, qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b[2], b[3]);
                }
                // this lane's keys: key0 + 2t, +1 (s0), +8, +9 (s1); elements 0, 1 of row g, 2, 3 of row g + 8
                uint32_t pa[4];
                float alpha[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float v[4] = {s0[2 * half], s0[2 * half + 1], s1[2 * half], s1[2 * half + 1]};
                    float top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        int key = key0 + 2 * t + (j & 1) + (j >> 1) * 8;
                        v[j] = key <= pos[half] ? v[j] * a.scale_log2 : -INFINITY;
                        top = fmaxf(top, v[j]);
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    float new_max = fmaxf(run_max[half], top), against = new_max == -INFINITY ? 0.f : new_max;
                    alpha[half] = fast_exp2(run_max[half] - against);
                    float p[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] = fast_exp2(v[j] - against);
                    run_sum[half] = run_sum[half] * alpha[half] + ((p[0] + p[1]) + (p[2] + p[3]));       // of this lane's keys
                    run_max[half] = new_max;
                    pa[half] = pack_bf16(p[0], p[1]);
                    pa[2 + half] = pack_bf16(p[2], p[3]);
                }
                if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {       // a maximum has moved
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) {
                        acc[n][0] *= alpha[0];
                        acc[n][1] *= alpha[0];
                        acc[n][2] *= alpha[1];
                        acc[n][3] *= alpha[1];
                    }
                }
                const bool cut = key0 + 15 > limit;          // values behind the last position are whatever the page held: zero here
                const int left = limit + 1 - key0 - 2 * t;   // of this lane's keys 0, 1, 8, 9
                const uint32_t keep_low = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
                const uint32_t keep_high = left >= 10 ? 0xffffffffu : left == 9 ? 0xffffu : 0u;
#pragma unroll
                for (int n = 0; n < HD / 8; n += 2) {
                    uint32_t b[4];
                    ldmatrix_x4_trans(b, swizzled(v_page, part * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), (n + (lane >> 4)) * 8));
                    if (cut) {
                        b[0] &= keep_low;
                        b[1] &= keep_high;
                        b[2] &= keep_low;
                        b[3] &= keep_high;
                    }
                    mma_bf16(acc[n], pa[0], pa[1], pa[2], pa[3], b[0], b[1]);
                    mma_bf16(acc[n + 1], pa[0], pa[1], pa[2], pa[3], b[2], b[3]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&empty[stage]));
        }
    }
    __syncthreads();                                         // every page has been read: its room is free
    if (*abort_flag) {                                       // a wait ran out: copies in flight get their time before the block leaves
        for (int i = 0; i < 100; ++i) __nanosleep(10000);
        if (a.behind) griddep_wait();
        return;
    }
    constexpr int LD = HD + 8;                               // (rows of the merge in different banks)
    float* merge_acc = reinterpret_cast<float*>(base);       // [warps][16][LD]
    float* merge_max = merge_acc + FEW_WARPS * 16 * LD;      // [warps][16], and the sums
    float* merge_sum = merge_max + FEW_WARPS * 16;
    if (warp < FEW_WARPS) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            run_sum[half] += __shfl_xor_sync(0xffffffffu, run_sum[half], 1);
            run_sum[half] += __shfl_xor_sync(0xffffffffu, run_sum[half], 2);
            int r = part * 16 + g + half * 8;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
                *reinterpret_cast<float2*>(merge_acc + r * LD + n * 8 + 2 * t) = make_float2(acc[n][2 * half], acc[n][2 * half + 1]);
            if (t == 0) {
                merge_max[r] = run_max[half];
                merge_sum[r] = run_sum[half];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < w.n_rows * (HD / 4); i += FEW_THREADS) {
        int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < FEW_WARPS; ++k) m = fmaxf(m, merge_max[k * 16 + r]);
        float against = m == -INFINITY ? 0.f : m, sum = 0.f;
        float4 value = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < FEW_WARPS; ++k) {
            float weight = fast_exp2(merge_max[k * 16 + r] - against);
            float4 x = *reinterpret_cast<const float4*>(merge_acc + (k * 16 + r) * LD + d);
            value.x = fmaf(x.x, weight, value.x);
            value.y = fmaf(x.y, weight, value.y);
            value.z = fmaf(x.z, weight, value.z);
            value.w = fmaf(x.w, weight, value.w);
            sum += merge_sum[k * 16 + r] * weight;
        }
        int token = w.first_token + r / share, head = w.kv_head * share + r % share;
        if (a.slots == 1) {
            float inv = sum != 0.f ? 1.f / sum : 0.f;
            uint2 packed = make_uint2(pack2(value.x * inv, value.y * inv), pack2(value.z * inv, value.w * inv));
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (size_t)token * a.out_stride + (size_t)head * HD + d) = packed;
        } else {
            size_t row = (size_t)token * a.n_heads + head;
            if (sum != 0.f) *reinterpret_cast<float4*>(a.acc + (row * a.slots + w.slot) * HD + d) = value;
            if (d == 0) put_stats(a, w, pieces, row, m, sum);
        }
    }
    if (a.behind) griddep_wait();
}

// Up to 128 rows over a group's shared pages [page_begin, page_end).
template <int HD>
__global__ void __launch_bounds__(TILE_THREADS, 2)
prefix_attention_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                             const __grid_constant__ Args args, int* status) {
    constexpr int PIECES = HD / 64, KV_BYTES = PIECES * KV_PIECE;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + Ring<HD>::BYTES);         // 15 barriers and two words
    unsigned char* q_tile = base;
    unsigned char* k_tile = base + PIECES * Q_PIECE;
    unsigned char* v_tile = k_tile + 2 * KV_BYTES;
    uint64_t* q_full = bars;                  // the queries are in shared memory
    uint64_t* k_full = bars + 1;              // [2]
    uint64_t* k_empty = bars + 3;             // [2]
    uint64_t* v_full = bars + 5;              // [2]
    uint64_t* v_empty = bars + 7;             // [2]
    uint64_t* s_full = bars + 9;              // [2] a buffer's scores are complete
    uint64_t* p_full = bars + 11;             // [2] its weights are written and O has been rescaled
    uint64_t* o_full = bars + 13;             // a page's P V has been added to O (asked for at the next page only: a parity tells two states apart)
    uint64_t* o_last = bars + 14;             // the last one's has
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = warp_index(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
#pragma unroll 1
        for (int i = 0; i < 15; ++i) mbar_init(smem_u32(&bars[i]), (i == 0 || i == 11 || i == 12) ? 128 : 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __shared__ Staged staged;
    Args a = args;
    stage_arrays(a, staged);
    Item w;
    int pieces;
    const bool work = slice_of(a, w, pieces, TC_ROWS, status);                // nothing is allocated where a block leaves
    const int share = a.n_heads / a.n_kv_heads, n_pages = work ? w.page_end - w.page_begin : 0;
    // Tensor memory is taken when the kernel in front is done with it, and the next kernel may take some only when this one has it: two
    // that wait for one another's would stand still.
    griddep_wait();
    if (n_pages <= 0) {                                      // a slice beyond the group's pages, where all groups are cut alike
        for (int r = threadIdx.x; work && r < w.n_rows; r += TILE_THREADS)
            put_stats(a, w, pieces, (size_t)(w.first_token + r / share) * a.n_heads + w.kv_head * share + r % share, -INFINITY, 0.f);
        return;
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    griddep_launch();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        const int* pages = a.block_table + (size_t)w.seq_first * a.table_stride + w.page_begin;
        int numbers = lane < n_pages ? pages[lane] : 0;      // 32 places of the table at once
        for (int kb = 0; kb < n_pages; ++kb) {
            const int b = kb & 1, phase = ((kb >> 1) - 1) & 1;
            if (kb > 0 && (kb & 31) == 0) numbers = kb + lane < n_pages ? pages[kb + lane] : 0;
            const int row = (__shfl_sync(0xffffffffu, numbers, kb & 31) * a.n_kv_heads + w.kv_head) * LLMB_PAGE;
            for (int of = 0; of < 2; ++of) {                 // keys, values
                if (kb >= 2 && !mbar_wait_warp(smem_u32(of ? &v_empty[b] : &k_empty[b]), phase, abort_flag, status, 11 + of)) break;
                if (elect_one()) {
                    uint32_t bar = smem_u32(of ? &v_full[b] : &k_full[b]);
                    mbar_expect_tx(bar, KV_BYTES);
                    for (int h = 0; h < PIECES; ++h)
                        tma_load_2d(smem_u32((of ? v_tile : k_tile) + b * KV_BYTES + h * KV_PIECE), of ? &map_v : &map_k, bar, h * 64, row);
                }
                __syncwarp();
            }
            if (*abort_flag) break;
        }
    } else if (warp == 1) {
        // D 32-bit, A and B bfloat16, M = 128; S has N = 64 keys, O has N = HD with B MN-major
        constexpr uint32_t idesc_qk = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(LLMB_PAGE >> 3) << 17) | ((uint32_t)(TC_ROWS >> 4) << 24);
        constexpr uint32_t idesc_pv = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(TC_ROWS >> 4) << 24);
        const uint64_t q_desc = smem_desc(smem_u32(q_tile));
        const uint64_t k_desc0 = smem_desc(smem_u32(k_tile)), v_desc0 = smem_desc_mn(smem_u32(v_tile), KV_PIECE);
        constexpr uint64_t BUFFER = (uint64_t)(KV_BYTES >> 4);       // the second buffer, in the address field
        auto issue_qk = [&](int kb) -> bool {
            int b = kb & 1;
            if (!mbar_wait_warp(smem_u32(&k_full[b]), (kb >> 1) & 1, abort_flag, status, 14)) return false;
            tcgen05_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int j = 0; j < HD / 16; ++j) {
                    uint64_t q_off = (uint64_t)(((j >> 2) * Q_PIECE + (j & 3) * 32) >> 4);
                    uint64_t k_off = (uint64_t)(((j >> 2) * KV_PIECE + (j & 3) * 32) >> 4);
                    tcgen05_mma(tmem_base + S_COL + b * LLMB_PAGE, q_desc + q_off, k_desc0 + b * BUFFER + k_off, idesc_qk, j > 0 ? 1u : 0u);
                }
                tcgen05_commit(smem_u32(&s_full[b]));
                tcgen05_commit(smem_u32(&k_empty[b]));
            }
            __syncwarp();
            return true;
        };
        bool ok = mbar_wait_warp(smem_u32(q_full), 0, abort_flag, status, 13) && issue_qk(0);
        if (ok && n_pages > 1) ok = issue_qk(1);
        for (int kb = 0; kb < n_pages && ok; ++kb) {
            int b = kb & 1, phase = (kb >> 1) & 1;
            ok = mbar_wait_warp(smem_u32(&p_full[b]), phase, abort_flag, status, 15);
            ok = ok && mbar_wait_warp(smem_u32(&v_full[b]), phase, abort_flag, status, 16);
            if (!ok) break;
            tcgen05_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int j = 0; j < LLMB_PAGE / 16; ++j)    // 16 keys a step: 8 columns of weights, 2048 bytes of value rows
                    tcgen05_mma_ts(tmem_base + O_COL, tmem_base + S_COL + b * LLMB_PAGE + j * 8,
                                   v_desc0 + b * BUFFER + (uint64_t)((j * 2048) >> 4), idesc_pv, (kb > 0 || j > 0) ? 1u : 0u);
                tcgen05_commit(smem_u32(kb == n_pages - 1 ? o_last : o_full));
                tcgen05_commit(smem_u32(&v_empty[b]));
            }
            __syncwarp();
            if (kb + 2 < n_pages) ok = issue_qk(kb + 2);
        }
    } else {
        constexpr int CHUNKS = HD / 8, STEP = 128 / CHUNKS;
        const int t = threadIdx.x - 64;                      // 0 .. 127
        {   // the queries, 16 bytes at a time, where the 128-byte swizzle has them
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q);
            const int c = t % CHUNKS, more_tokens = STEP / share, more_heads = STEP % share;
            int token0 = w.first_token + t / CHUNKS / share, head0 = t / CHUNKS % share;
#pragma unroll 1
            for (int r = t / CHUNKS; r < TC_ROWS; r += STEP) {
                unsigned char* chunk = q_tile + (c >> 3) * Q_PIECE + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                if (r < w.n_rows) cp_async16(chunk, q + (size_t)token0 * a.q_stride + (size_t)(w.kv_head * share + head0) * HD + c * 8);
                else *reinterpret_cast<uint4*>(chunk) = make_uint4(0u, 0u, 0u, 0u);
                token0 += more_tokens;
                head0 += more_heads;
                if (head0 >= share) {
                    head0 -= share;
                    ++token0;
                }
            }
            cp_async_commit();
        }
        const int quarter = warp & 3, row = quarter * 32 + lane;             // row of the tile = lane of tensor memory
        const int token = w.first_token + min(row, w.n_rows - 1) / share;
        const int my_pos = row < w.n_rows ? position_of(a, w, token) : -1;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const bool idle = quarter * 32 >= w.n_rows;          // a warp without rows: its lanes' weights reach nobody's result
        float run_max = -INFINITY, run_sum = 0.f;
        cp_async_wait<0>();
        fence_async_shared();
        mbar_arrive(smem_u32(q_full));
        bool ok = true;
        for (int kb = 0; kb < n_pages && ok; ++kb) {
            const int b = kb & 1, pos = my_pos - (w.page_begin + kb) * LLMB_PAGE;        // the last key that the row sees, from the page's first
            ok = mbar_wait_warp(smem_u32(&s_full[b]), (kb >> 1) & 1, abort_flag, status, 17);      // one answer for the warp: its loads are the whole warp's
            if (!ok) break;
            if (idle) {
                mbar_arrive(smem_u32(&p_full[b]));
                continue;
            }
            tcgen05_fence_after();
            const uint32_t s_addr = lane_addr + S_COL + b * LLMB_PAGE;
            uint32_t ra[32], rb[32];
            tmem_ld32_start(s_addr, ra);
            tmem_ld32_start(s_addr + 32, rb);
            tmem_ld32_wait(ra);
            tmem_ld32_wait(rb);
            if (pos < LLMB_PAGE - 1) {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    if (j > pos) ra[j] = __float_as_uint(-INFINITY);
                    if (j + 32 > pos) rb[j] = __float_as_uint(-INFINITY);
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 32; j += 2) top = max3(top, __uint_as_float(ra[j]), __uint_as_float(ra[j + 1]));
#pragma unroll
            for (int j = 0; j < 32; j += 2) top = max3(top, __uint_as_float(rb[j]), __uint_as_float(rb[j + 1]));
            // The maximum that the exponents refer to moves only when it is exceeded by more than 2^8; a row that has seen no key keeps -inf.
            const bool move = (top - run_max) * a.scale_log2 > 8.f;
            const float new_max = move ? top : run_max;
            const float alpha = move && kb > 0 ? fast_exp2((run_max - new_max) * a.scale_log2) : 1.f;
            const float shift = new_max == -INFINITY ? 0.f : new_max * a.scale_log2;
            run_max = new_max;
            float add = 0.f;
            auto to_weights = [&](const uint32_t (&x)[32], int c) {
                uint32_t packed[16];
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    float p0 = fast_exp2(fmaf(__uint_as_float(x[j]), a.scale_log2, -shift));
                    float p1 = fast_exp2(fmaf(__uint_as_float(x[j + 1]), a.scale_log2, -shift));
                    add += p0 + p1;
                    packed[j >> 1] = pack2(p0, p1);
                }
                tmem_st16(s_addr + (c >> 1), packed);
            };
            to_weights(ra, 0);
            to_weights(rb, 32);
            run_sum = run_sum * alpha + add;
            if (kb > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                ok = mbar_wait_warp(smem_u32(o_full), (kb - 1) & 1, abort_flag, status, 18);
                if (!ok) break;
                tcgen05_fence_after();
#pragma unroll 1
                for (int c = 0; c < HD; c += 16) {
                    uint32_t x[16];
                    tmem_ld16(lane_addr + O_COL + c, x);
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * alpha);
                    tmem_st16(lane_addr + O_COL + c, x);
                }
            }
            tmem_st_wait();
            tcgen05_fence_before();
            mbar_arrive(smem_u32(&p_full[b]));
        }
        if (ok) ok = mbar_wait_warp(smem_u32(o_last), 0, abort_flag, status, 19);
        if (ok && !idle) {
            tcgen05_fence_after();
            // All products are complete, the pages' room is free: a row goes out from there in one bulk copy. Rows lie 16 bytes further
            // apart than they are long.
            constexpr int ROOM = HD * 4 + 16;
            static_assert(TC_ROWS * ROOM <= Ring<HD>::BYTES, "a row a thread");
            unsigned char* room = base + row * ROOM;
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
                uint32_t x[16];
                tmem_ld16(lane_addr + O_COL + c, x);
#pragma unroll
                for (int d = 0; d < 16; d += 4) *reinterpret_cast<uint4*>(room + (c + d) * 4) = make_uint4(x[d], x[d + 1], x[d + 2], x[d + 3]);
            }
            if (row < w.n_rows) {
                const size_t at = (size_t)token * a.n_heads + w.kv_head * share + row % share;
                put_stats(a, w, pieces, at, run_max * a.scale_log2, run_sum);
                fence_async_shared();
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                             ::"l"(a.acc + (at * a.slots + w.slot) * HD), "r"(smem_u32(room)), "r"(HD * 4) : "memory");
                bulk_commit();
                bulk_wait<0>();
            }
        }
    }

    tcgen05_fence_before();
    __syncthreads();
    if (*abort_flag) {                                       // a wait ran out: copies in flight get their time before the block leaves
        for (int i = 0; i < 100; ++i) __nanosleep(10000);
        __syncthreads();
    }
    if (warp == 1) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

// ------------------------------------------------------------------------------------------------ bfloat16, many rows
//
// 256 rows a block, one block an SM: two tiles of 128 rows with four softmax warps each share the keys and values of 128 positions (two
// pages). Per tile one buffer of scores [128, 128] and O [128, D] fill tensor memory; the two tiles take turns: while the softmax of one
// works on its scores, the products of the other run (P V of these keys, then Q K^T of the next). Against two blocks an SM of 128 rows and 64 keys
// each step has half the waits per score, Q K^T reads 8 KB of shared memory for 64 cycles of products (with 64 keys 6 KB for 32: the
// reads, not the products, set its pace), and every page is read once for 256 rows.
//
// When a tile's scores are there, its last P V is complete too (the products were issued behind it), so O can be rescaled at once. The maximum
// that the exponents refer to moves only when it is exceeded by more than 2^8. Weights are rounded to 8 bits, what the tensor cores
// take; their sum is of the unrounded ones.
//
// A walk is a group's shared pages and, where the sequences bring many tokens (`whole`), behind them the own pages of each sequence that the
// block has rows of. Only the rows of that sequence see those: the others' weights are zero, and the products leave their lanes of O
// alone (a value that is not finite times a weight of zero would reach them).

constexpr int WIDE_THREADS = 384;           // warps 0 keys, 1 products, 2 values, 4-7 and 8-11 a tile's softmax
constexpr int PAIR_PIECE = 128 * 128;                        // 128 positions, 64 columns of the head: 16 KB
// of the warps that issue and of the softmax's (64 and 216 spilled in the loop that issues)
constexpr int WIDE_REGS_FEW = 104, WIDE_REGS_MANY = 200, WIDE_REGS_LAUNCHED = 168;
static_assert(128 * WIDE_REGS_FEW + 256 * WIDE_REGS_MANY <= WIDE_THREADS * WIDE_REGS_LAUNCHED, "the shares come from what the block is launched with");

// The pages of an item, one after the other: the shared ones, then those of each sequence in turn.
struct Walk {
    int seq;                          // whose own pages these are, or -1 for shared ones
    int logical, end;                 // place in the table of the sequence (of the first one where shared), end of this stretch
    int limit;                        // the last position of the stretch that a row of the tile sees
};

// the tile's rows are tokens first .. last of sequences seq_first .. seq_last
struct TileRange {
    int seq_first, seq_last, token_first, token_last, shared;
    bool own;                         // own pages behind the shared ones
};

__device__ __forceinline__ void own_stretch(const Args& a, const TileRange& t, int seq, Walk& w) {
    w.seq = seq;
    int end = a.cu_seqlens[seq + 1];
    w.limit = a.seq_lens[seq] - end + min(end - 1, t.token_last);         // position of the sequence's last token in the tile
    w.logical = t.shared;
    w.end = w.limit / LLMB_PAGE + 1;
    if (a.cu_seqlens[seq] == end || w.limit < 0) w.end = 0;                 // brings nothing
}
__device__ __forceinline__ bool next_stretch(const Args& a, const TileRange& t, Walk& w) {
    while (t.own) {
        int seq = w.seq < 0 ? t.seq_first : w.seq + 1;
        if (seq > t.seq_last) return false;
        own_stretch(a, t, seq, w);
        if (w.logical < w.end) return true;
    }
    return false;
}
__device__ __forceinline__ bool step(const Args& a, const TileRange& t, Walk& w) { return ++w.logical < w.end || next_stretch(a, t, w); }
// to the page `skip` pages behind the walk's first
__device__ __forceinline__ void start(const Args& a, const TileRange& t, Walk& w, int skip) {
    w.seq = -1;
    w.logical = 0;
    w.end = t.shared;
    w.limit = t.shared * LLMB_PAGE - 1;
    while (skip >= w.end - w.logical) {
        skip -= max(w.end - w.logical, 0);
        if (!next_stretch(a, t, w)) return;
    }
    w.logical += skip;
}

// a block's tile, its piece of the tile's walk, and how many pieces that has
struct Piece {
    int kv_head, group, tile, tile_index, piece, pieces;
};
// Every tile is cut alike (`whole`, and batches too large for the arrays in shared memory).
__device__ __forceinline__ Piece piece_of(const Args& a, int x) {
    Piece p{0, 0, 0, x, 0, 1};
    if (x >= a.full_tiles) {
        x -= a.full_tiles;
        p.tile_index = a.full_tiles + x / a.prefix_splits;
        p.piece = x % a.prefix_splits;
        p.pieces = a.prefix_splits;
    }
    int rest = p.tile_index / a.n_kv_heads;
    p.kv_head = p.tile_index - rest * a.n_kv_heads;
    p.group = rest / a.prefix_tiles;
    p.tile = rest - p.group * a.prefix_tiles;
    return p;
}
// Groups of unequal lengths: pieces of `per` pairs of pages, the least number with which all tiles' pieces fit into the grid. Each warp finds out
// for itself, a lane a group. group = n_groups where nothing is left for the block.
__device__ __forceinline__ Piece even_piece_of(const Args& a, int x, int blocks, int lane) {
    const unsigned all = 0xffffffffu;
    const int share = a.n_heads / a.n_kv_heads, heads = blocks / a.n_kv_heads;      // blocks of a key head
    auto tiles_and_pairs = [&](int g, int& tiles, int& pairs) {
        tiles = 0;
        pairs = 0;
        if (g < a.n_groups) {
            tiles = ((a.cu_seqlens[a.group_first[g + 1]] - a.cu_seqlens[a.group_first[g]]) * share + WIDE_ROWS - 1) / WIDE_ROWS;
            pairs = (a.group_pages[g] + 1) / 2;
            if (pairs == 0 || tiles < 0) tiles = 0;
        }
    };
    int work = 0, items = 0, most = 0, tiles, pairs;
    for (int g0 = 0; g0 < a.n_groups; g0 += 32) {
        tiles_and_pairs(g0 + lane, tiles, pairs);
        work += __reduce_add_sync(all, tiles * pairs);
        items += __reduce_add_sync(all, tiles);
        most = max(most, __reduce_max_sync(all, tiles > 0 ? pairs : 0));
    }
    int per = items < heads ? (work + heads - items - 1) / (heads - items) : most;
    per = max(max(per, (most + a.prefix_splits - 1) / a.prefix_splits), 1);
    Piece p{x % a.n_kv_heads, a.n_groups, 0, 0, 0, 1};
    x /= a.n_kv_heads;
    for (int g0 = 0; g0 < a.n_groups; g0 += 32) {
        tiles_and_pairs(g0 + lane, tiles, pairs);
        int pieces = (pairs + per - 1) / per, before = tiles * pieces;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            int left = __shfl_up_sync(all, before, d);
            if (lane >= d) before += left;
        }
        unsigned beyond = __ballot_sync(all, x < before);
        if (beyond) {
            int at = __ffs(beyond) - 1;
            p.group = g0 + at;
            p.pieces = __shfl_sync(all, pieces, at);
            x -= __shfl_sync(all, before - tiles * pieces, at);
            p.tile = x / p.pieces;
            p.piece = x - p.tile * p.pieces;
            break;
        }
        x -= __shfl_sync(all, before, 31);
    }
    return p;
}

// A from tensor memory, B from shared memory; lanes whose bit is set in `off` keep their rows of D
__device__ __forceinline__ void mma_ts_lanes(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, const uint32_t (&off)[4]) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(1u), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3]) : "memory");
}
// the lanes of a tile that are not among rows first .. last - 1
__device__ __forceinline__ void lanes_off(int first, int last, uint32_t (&off)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        int from = min(max(first - 32 * k, 0), 32), to = min(max(last - 32 * k, 0), 32);
        uint32_t below_to = to >= 32 ? 0xffffffffu : (1u << to) - 1u, below_from = from >= 32 ? 0xffffffffu : (1u << from) - 1u;
        off[k] = ~(below_to & ~below_from);
    }
}

template <int HD>
__global__ void __launch_bounds__(WIDE_THREADS, 1)
prefix_attention_wide_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                             const __grid_constant__ Args args, int* status) {
    constexpr int PIECES = HD / 64;
    constexpr int Q_BYTES = PIECES * Q_PIECE, PAIR_BYTES = PIECES * PAIR_PIECE, PAGE_BYTES = PIECES * KV_PIECE;
    constexpr uint32_t SCORES = 128, O_FIRST = 256, COLS = 512;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* q_tile = base;                             // [2]
    unsigned char* k_tile = base + 2 * Q_BYTES;               // [2] pairs of pages
    unsigned char* v_tile = k_tile + 2 * PAIR_BYTES;          // [2]
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_tile + 2 * PAIR_BYTES);
    uint64_t* q_full = bars;                  // [2] a tile's queries are in shared memory
    uint64_t* k_full = bars + 2;              // [2]
    uint64_t* k_empty = bars + 4;             // [2]
    uint64_t* v_full = bars + 6;              // [2]
    uint64_t* v_empty = bars + 8;             // [2]
    uint64_t* s_full = bars + 10;             // [2] a tile's scores are complete (and all its products before)
    uint64_t* p_full = bars + 12;             // [2][2] its weights of 64 positions are written and O has been rescaled
    uint64_t* o_full = bars + 16;             // [2] its last P V is complete
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    __shared__ Staged staged;
    Args a = args;
    stage_arrays(a, staged);
    const Piece piece = a.even_blocks ? even_piece_of(a, blockIdx.x, gridDim.x, threadIdx.x & 31) : piece_of(a, blockIdx.x);
    const int share = a.n_heads / a.n_kv_heads;
    Item w;
    w.kv_head = piece.kv_head;
    w.tile = piece.tile;
    const int group = piece.group;
    // A block without work leaves here (the block as a whole, nothing is allocated yet), behind the kernel in front all the same: if
    // none has any (a step whose groups turn out to share nothing), the own parts that follow rely on these waits alone.
    if (group >= a.n_groups) return griddep_wait();
    w.seq_first = a.group_first[group];
    w.seq_last = a.group_first[group + 1];
    if (w.seq_first >= w.seq_last) return griddep_wait();
    w.first_token = a.cu_seqlens[w.seq_first];
    w.n_rows = (a.cu_seqlens[w.seq_last] - w.first_token) * share;
    if (w.n_rows > a.prefix_tiles * WIDE_ROWS) report_beyond_bounds(status);       // (tiles that no block has)
    const int row0 = w.tile * WIDE_ROWS, n_rows = min(WIDE_ROWS, w.n_rows - row0);
    if (n_rows <= 0) return griddep_wait();
    const int n_tiles = n_rows > TC_ROWS ? 2 : 1;
    TileRange range;
    range.token_first = w.first_token + row0 / share;
    range.token_last = w.first_token + (row0 + n_rows - 1) / share;
    range.seq_first = sequence_of(a, w, range.token_first);
    range.seq_last = sequence_of(a, w, range.token_last);
    range.own = a.whole;
    range.shared = a.group_pages[group];
    int total = range.shared;
    if (a.whole) {
        Walk all;
        all.seq = -1;
        while (next_stretch(a, range, all)) total += all.end - all.logical;
    }
    // pieces of whole pairs of pages
    const int pairs = (total + 1) / 2, per = (pairs + piece.pieces - 1) / piece.pieces;
    const int skip = min(piece.piece * per * 2, total), n_pages = min(per * 2, total - skip), n_blocks = (n_pages + 1) / 2;
    const int* shared_pages = a.block_table + (size_t)w.seq_first * a.table_stride;
    const int warp = warp_index(), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
#pragma unroll 1
        for (int i = 0; i < 18; ++i) {
            bool by_softmax = i < 2 || (i >= 12 && i < 16);
            mbar_init(smem_u32(&bars[i]), by_softmax ? 128 : 1);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Tensor memory is taken when the kernel in front is done with it, and the next kernel may take some only when this one has it: two
    // that wait for one another's would stand still.
    griddep_wait();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    griddep_launch();
    uint32_t tmem_base = *tmem_slot;

    // page i of the piece: shared ones first, then what the walk finds behind them
    struct Place {
        int seq, logical, limit;
    };
    const int n_shared = max(0, min(n_pages, range.shared - skip));
    Walk walk;
    if (n_shared < n_pages) start(a, range, walk, skip + n_shared);
    auto next_place = [&](int i) -> Place {
        if (i < n_shared) return Place{-1, skip + i, 0x7fffffff};
        Place at{walk.seq, walk.logical, walk.limit};
        step(a, range, walk);
        return at;
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(WIDE_REGS_FEW));
        if (warp == 0 || warp == 2) {
            const bool keys = warp == 0;
            const CUtensorMap* map = keys ? &map_k : &map_v;
            unsigned char* tiles = keys ? k_tile : v_tile;
            uint64_t* full = keys ? k_full : v_full;
            uint64_t* empty = keys ? k_empty : v_empty;
            auto next_page = [&](int i) {
                Place at = next_place(i);
                return (at.seq < 0 ? shared_pages : a.block_table + (size_t)at.seq * a.table_stride)[at.logical];
            };
            int first = n_pages > 0 ? next_page(0) : 0, second = n_pages > 1 ? next_page(1) : -1;
            for (int kb = 0; kb < n_blocks; ++kb) {
                int b = kb & 1, page0 = first, page1 = second;
                // the numbers of the next pages are fetched under the wait for room
                if (2 * kb + 2 < n_pages) first = next_page(2 * kb + 2);
                second = 2 * kb + 3 < n_pages ? next_page(2 * kb + 3) : -1;
                if (kb >= 2 && !mbar_wait_warp(smem_u32(&empty[b]), ((kb >> 1) - 1) & 1, abort_flag, status, keys ? 31 : 32)) break;
                if (elect_one()) {
                    uint32_t bar = smem_u32(&full[b]);
                    mbar_expect_tx(bar, page1 >= 0 ? 2 * PAGE_BYTES : PAGE_BYTES);
                    for (int h = 0; h < PIECES; ++h) {
                        uint32_t to = smem_u32(tiles + b * PAIR_BYTES + h * PAIR_PIECE);
                        tma_load_2d(to, map, bar, h * 64, (page0 * a.n_kv_heads + w.kv_head) * LLMB_PAGE);
                        if (page1 >= 0) tma_load_2d(to + KV_PIECE, map, bar, h * 64, (page1 * a.n_kv_heads + w.kv_head) * LLMB_PAGE);
                    }
                }
                __syncwarp();
            }
        } else if (warp == 1) {
            // The tiles' products in turn, which keeps them half a period apart: with a warp for each both softmaxes ran at the same time
            // and shared the special-function units while the tensor cores stood still (4,350 cycles a pair of pages).
            constexpr uint32_t idesc_qk = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(TC_ROWS >> 4) << 24);
            constexpr uint32_t idesc_pv = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(TC_ROWS >> 4) << 24);
            const uint64_t q_desc = smem_desc(smem_u32(q_tile));
            const uint64_t k_desc0 = smem_desc(smem_u32(k_tile)), v_desc0 = smem_desc_mn(smem_u32(v_tile), PAIR_PIECE);
            constexpr uint64_t BUFFER = (uint64_t)(PAIR_BYTES >> 4), Q_TILE = (uint64_t)(Q_BYTES >> 4);
            auto issue_qk = [&](int tile, int kb) {
                int b = kb & 1;
                if (elect_one()) {
#pragma unroll
                    for (int j = 0; j < HD / 16; ++j) {
                        uint64_t q_off = (uint64_t)(((j >> 2) * Q_PIECE + (j & 3) * 32) >> 4);
                        uint64_t k_off = (uint64_t)(((j >> 2) * PAIR_PIECE + (j & 3) * 32) >> 4);
                        tcgen05_mma(tmem_base + tile * SCORES, q_desc + tile * Q_TILE + q_off, k_desc0 + b * BUFFER + k_off, idesc_qk, j > 0 ? 1u : 0u);
                    }
                    tcgen05_commit(smem_u32(&s_full[tile]));
                    if (tile == n_tiles - 1) tcgen05_commit(smem_u32(&k_empty[b]));
                }
                __syncwarp();
            };
            // the values of pair kb and the keys of the pair behind it are in shared memory
            auto arrived = [&](int kb) {
                return mbar_wait_warp(smem_u32(&v_full[kb & 1]), (kb >> 1) & 1, abort_flag, status, 36) &&
                       (kb + 1 >= n_blocks || mbar_wait_warp(smem_u32(&k_full[(kb + 1) & 1]), ((kb + 1) >> 1) & 1, abort_flag, status, 37));
            };
            bool ok = n_blocks > 0 && mbar_wait_warp(smem_u32(&k_full[0]), 0, abort_flag, status, 34);
            for (int tile = 0; tile < n_tiles && ok; ++tile) {
                ok = mbar_wait_warp(smem_u32(&q_full[tile]), 0, abort_flag, status, 33);
                if (!ok) break;
                tcgen05_fence_after();
                issue_qk(tile, 0);
            }
            ok = ok && arrived(0);
            // A tile's products of pair kb, then its scores of the next pair. `masked`: pages that not all rows of the tile may be touched by, or a
            // single page at the end; otherwise nothing is worked out between the waits (the tensor cores have work for some 500 cycles).
            auto turn = [&](int tile, int kb, bool masked, bool two, const uint32_t (&off)[2][4]) -> bool {
                const int b = kb & 1;
                const uint32_t o = tmem_base + O_FIRST + tile * HD, p = tmem_base + tile * SCORES;
#pragma unroll
                for (int half = 0; half < 2; ++half) {        // 64 positions each: the first are multiplied while the others' weights are formed
                    if (!mbar_wait_warp(smem_u32(&p_full[2 * tile + half]), kb & 1, abort_flag, status, 35)) return false;
                    tcgen05_fence_after();
                    // 16 positions a step: 8 columns of weights, 2048 bytes of value rows
                    if (!masked) {
                        if (elect_one()) {
#pragma unroll
                            for (int j = 4 * half; j < 4 * half + 4; ++j)
                                tcgen05_mma_ts(o, p + j * 8, v_desc0 + b * BUFFER + (uint64_t)((j * 2048) >> 4), idesc_pv, 1u);
                        }
                    } else if ((half == 0 || two) && elect_one()) {
#pragma unroll
                        for (int j = 4 * half; j < 4 * half + 4; ++j)
                            mma_ts_lanes(o, p + j * 8, v_desc0 + b * BUFFER + (uint64_t)((j * 2048) >> 4), idesc_pv, off[half]);
                    }
                    __syncwarp();
                }
                if (elect_one()) {
                    if (kb == n_blocks - 1) tcgen05_commit(smem_u32(&o_full[tile]));
                    if (tile == n_tiles - 1) tcgen05_commit(smem_u32(&v_empty[b]));
                }
                __syncwarp();
                if (kb + 1 < n_blocks) {
                    issue_qk(tile, kb + 1);
                    // the next keys and values are waited for where products are under way
                    if (tile == 0) return arrived(kb + 1);
                }
                return true;
            };
            // the rows of a tile that do not see a page, where the block has rows of several sequences
            const bool mixed = range.seq_first != range.seq_last;
            const int n_plain = mixed ? n_shared / 2 : n_pages / 2;              // pairs that every row may be touched by
            uint32_t none[2][4] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
            int kb = 0;
            if (n_tiles == 2) {
                for (; kb < n_plain && ok; ++kb) ok = turn(0, kb, false, true, none) && turn(1, kb, false, true, none);
            } else {
                for (; kb < n_plain && ok; ++kb) ok = turn(0, kb, false, true, none);
            }
            for (; kb < n_blocks && ok; ++kb) {
                const bool two = 2 * kb + 1 < n_pages;
                Place at[2];
                at[0] = next_place(2 * kb);
                if (two) at[1] = next_place(2 * kb + 1);
                for (int tile = 0; tile < n_tiles && ok; ++tile) {
                    uint32_t off[2][4] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if ((half && !two) || !mixed || at[half].seq < 0) continue;
                        lanes_off((a.cu_seqlens[at[half].seq] - w.first_token) * share - row0 - tile * TC_ROWS,
                                  (a.cu_seqlens[at[half].seq + 1] - w.first_token) * share - row0 - tile * TC_ROWS, off[half]);
                    }
                    ok = turn(tile, kb, true, two, off);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(WIDE_REGS_MANY));
        const int tile = (warp >> 2) - 1, quarter = warp & 3, t = threadIdx.x & 127;
        const int tile_rows = n_rows - tile * TC_ROWS;        // of this tile, above 128 where it is full
        if (tile < n_tiles) {
            constexpr int CHUNKS = HD / 8;
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q);
            unsigned char* to = q_tile + tile * Q_BYTES;
            // All 16-byte chunks in flight at once, and no division for each (the queries took 11,000 to 18,000 cycles with both).
            constexpr int STEP = 128 / CHUNKS;
            const int c = t % CHUNKS, at0 = row0 + tile * TC_ROWS + t / CHUNKS, more_tokens = STEP / share, more_heads = STEP % share;
            int token0 = w.first_token + at0 / share, head0 = at0 % share;
#pragma unroll 1
            for (int k = 0; k < CHUNKS; ++k) {
                int r = t / CHUNKS + k * STEP;
                unsigned char* chunk = to + (c >> 3) * Q_PIECE + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                const __nv_bfloat16* from = q + (size_t)token0 * a.q_stride + (size_t)(w.kv_head * share + head0) * HD + c * 8;
                token0 += more_tokens;
                head0 += more_heads;
                if (head0 >= share) {
                    head0 -= share;
                    ++token0;
                }
                if (r < tile_rows) {
                    cp_async16(chunk, from);
                } else {
                    *reinterpret_cast<uint4*>(chunk) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            cp_async_commit();

            // what a row needs besides, while the queries are on their way
            const int r = quarter * 32 + lane;                // row of the tile = lane of tensor memory
            const bool valid = r < tile_rows;
            const int at = row0 + tile * TC_ROWS + (valid ? r : 0);
            const int token = w.first_token + at / share, head = w.kv_head * share + at % share;
            const int my_seq = sequence_of(a, w, token);
            const int my_pos = valid ? a.seq_lens[my_seq] - a.cu_seqlens[my_seq + 1] + token : -1;
            const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
            const uint32_t s_addr = lane_addr + tile * SCORES, o_addr = lane_addr + O_FIRST + tile * HD;
            const bool idle = quarter * 32 >= tile_rows;      // a warp without rows: its lanes' weights reach nobody's result
            {   // every product adds to O: it starts from zero
                uint32_t zero[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) zero[j] = 0u;
#pragma unroll 1
                for (int c = 0; c < HD; c += 16) tmem_st16(o_addr + c, zero);
                tmem_st_wait();
            }
            cp_async_wait<0>();
            fence_async_shared();
            mbar_arrive(smem_u32(&q_full[tile]));
            const uint64_t scale2 = pair_of(a.scale_log2, a.scale_log2);
            float run_max = -INFINITY, run_sum = 0.f;
            bool ok = true;
            for (int kb = 0; kb < n_blocks && ok; ++kb) {
                // the last key that the row sees of each of the two pages, from the page's first; positions stored behind it that no row sees
                int pos0 = my_pos - (skip + 2 * kb) * LLMB_PAGE, pos1 = pos0 - LLMB_PAGE, stored0 = LLMB_PAGE, stored1 = LLMB_PAGE;
                if (2 * kb + 1 >= n_shared) {
                    Place at = next_place(2 * kb);
                    pos0 = (at.seq < 0 || at.seq == my_seq ? my_pos : -1) - at.logical * LLMB_PAGE;
                    stored0 = min(at.limit - at.logical * LLMB_PAGE, LLMB_PAGE - 1) + 1;
                    pos1 = -1;
                    if (2 * kb + 1 < n_pages) {
                        at = next_place(2 * kb + 1);
                        pos1 = (at.seq < 0 || at.seq == my_seq ? my_pos : -1) - at.logical * LLMB_PAGE;
                        stored1 = min(at.limit - at.logical * LLMB_PAGE, LLMB_PAGE - 1) + 1;
                    }
                }
                ok = mbar_wait_warp(smem_u32(&s_full[tile]), kb & 1, abort_flag, status, 38);
                if (!ok) break;
                tcgen05_fence_after();
                if (stored0 < LLMB_PAGE || stored1 < LLMB_PAGE) {     // values behind the last position are whatever a page held: zero here
                    ok = mbar_wait_warp(smem_u32(&v_full[kb & 1]), (kb >> 1) & 1, abort_flag, status, 39);
                    if (!ok) break;
                    for (int half = 0; half < 2 && tile == 0; ++half) {       // (the first tile's products are issued first)
                        int first = max(half ? stored1 : stored0, 0), chunks = (LLMB_PAGE - first) * 8;
                        for (int i = t; i < PIECES * chunks; i += 128) {
                            int h = i / chunks, rest = i - h * chunks;
                            *reinterpret_cast<uint4*>(v_tile + (kb & 1) * PAIR_BYTES + h * PAIR_PIECE + half * KV_PIECE + first * 128 + rest * 16) =
                                make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                    fence_async_shared();
                }
                if (idle) {
                    mbar_arrive(smem_u32(&p_full[2 * tile]));
                    mbar_arrive(smem_u32(&p_full[2 * tile + 1]));
                } else {
                    uint32_t r0[32], r1[32], r2[32], r3[32];
                    // the second half of the scores comes while the first one's maximum is taken
                    tmem_ld32_start(s_addr, r0);
                    tmem_ld32_start(s_addr + 32, r1);
                    tmem_ld32_wait(r0);
                    tmem_ld32_wait(r1);
                    tmem_ld32_start(s_addr + 64, r2);
                    tmem_ld32_start(s_addr + 96, r3);
                    if (pos0 < LLMB_PAGE - 1) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            if (j > pos0) r0[j] = __float_as_uint(-INFINITY);
                            if (j + 32 > pos0) r1[j] = __float_as_uint(-INFINITY);
                        }
                    }
                    float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        top0 = max3(top0, __uint_as_float(r0[j]), __uint_as_float(r0[j + 1]));
                        top1 = max3(top1, __uint_as_float(r1[j]), __uint_as_float(r1[j + 1]));
                    }
                    tmem_ld32_wait(r2);
                    tmem_ld32_wait(r3);
                    if (pos1 < LLMB_PAGE - 1) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            if (j > pos1) r2[j] = __float_as_uint(-INFINITY);
                            if (j + 32 > pos1) r3[j] = __float_as_uint(-INFINITY);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        top0 = max3(top0, __uint_as_float(r2[j]), __uint_as_float(r2[j + 1]));
                        top1 = max3(top1, __uint_as_float(r3[j]), __uint_as_float(r3[j + 1]));
                    }
                    const float top = fmaxf(top0, top1);
                    // (a row that has seen no key yet keeps -inf, and all its weights are zero)
                    const bool move = (top - run_max) * a.scale_log2 > 8.f;
                    const float new_max = move ? top : run_max;
                    const float alpha = move ? fast_exp2((run_max - new_max) * a.scale_log2) : 1.f;
                    const float shift = new_max == -INFINITY ? 0.f : -new_max * a.scale_log2;
                    run_max = new_max;
                    if (kb > 0 && __any_sync(0xffffffffu, move)) {
#pragma unroll 1
                        for (int c = 0; c < HD; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(o_addr + c, o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                            tmem_st16(o_addr + c, o);
                        }
                    }
                    const uint64_t shift2 = pair_of(shift, shift);
                    uint64_t add = pair_of(0u, 0u);
                    auto to_weights = [&](const uint32_t (&x)[32], int c) {
                        uint32_t packed[16];
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            float p0, p1;
                            unpair(fma2(pair_of(x[j], x[j + 1]), scale2, shift2), p0, p1);
                            p0 = fast_exp2(p0);
                            p1 = fast_exp2(p1);
                            add = add2(add, pair_of(p0, p1));
                            packed[j >> 1] = pack2(p0, p1);
                        }
                        tmem_st16(s_addr + (c >> 1), packed);
                    };
                    to_weights(r0, 0);
                    to_weights(r1, 32);
                    tmem_st_wait();
                    tcgen05_fence_before();
                    mbar_arrive(smem_u32(&p_full[2 * tile]));
                    to_weights(r2, 64);
                    to_weights(r3, 96);
                    float add_lo, add_hi;
                    unpair(add, add_lo, add_hi);
                    run_sum = run_sum * alpha + (add_lo + add_hi);
                    tmem_st_wait();
                    tcgen05_fence_before();
                    mbar_arrive(smem_u32(&p_full[2 * tile + 1]));
                }
            }
            // both tiles' products are complete: the pages' room is free
            for (int i = 0; i < n_tiles && ok && n_blocks > 0; ++i) ok = mbar_wait_warp(smem_u32(&o_full[i]), 0, abort_flag, status, 40);
            if (ok && !idle) {
                tcgen05_fence_after();
                const bool direct = piece.pieces == 1 && a.whole;
                const float inv = run_sum != 0.f ? 1.0f / run_sum : 0.f;
                const size_t part_row = a.whole ? (size_t)(piece.tile_index - a.full_tiles) * WIDE_ROWS + (at - row0) : (size_t)token * a.n_heads + head;
                const size_t slot = part_row * a.slots + piece.piece;
                if (valid && !direct) *reinterpret_cast<float2*>(a.stats + slot * 2) = make_float2(run_sum != 0.f ? run_max * a.scale_log2 : -INFINITY, run_sum);
                if (valid && a.even_blocks && piece.piece == piece.pieces - 1)           // the parts that this tile has fewer than others
                    for (int i = piece.pieces; i < a.prefix_splits; ++i)
                        *reinterpret_cast<float2*>(a.stats + (part_row * a.slots + i) * 2) = make_float2(-INFINITY, 0.f);
                // O goes out by way of shared memory, a bulk copy a row: written from its thread, a row's 16 bytes each went to another line
                // (9,000 to 15,000 cycles). Rows lie 16 bytes further apart than they are long: eight lanes' chunks in different banks.
                constexpr int ROOM = HD * 4 + 16;
                static_assert(2 * TC_ROWS * ROOM <= 2 * Q_BYTES + 4 * PAIR_BYTES, "rows of both tiles");
                unsigned char* room = base + (tile * TC_ROWS + r) * ROOM;
                if (direct || n_blocks > 0) {
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t x[32];
                        tmem_ld32(o_addr + c, x);
                        if (direct) {
#pragma unroll
                            for (int d = 0; d < 32; d += 8)
                                *reinterpret_cast<uint4*>(room + (c + d) * 2) = make_uint4(
                                    pack2(__uint_as_float(x[d]) * inv, __uint_as_float(x[d + 1]) * inv), pack2(__uint_as_float(x[d + 2]) * inv, __uint_as_float(x[d + 3]) * inv),
                                    pack2(__uint_as_float(x[d + 4]) * inv, __uint_as_float(x[d + 5]) * inv), pack2(__uint_as_float(x[d + 6]) * inv, __uint_as_float(x[d + 7]) * inv));
                        } else {
#pragma unroll
                            for (int d = 0; d < 32; d += 4) *reinterpret_cast<uint4*>(room + (c + d) * 4) = make_uint4(x[d], x[d + 1], x[d + 2], x[d + 3]);
                        }
                    }
                    if (valid) {
                        fence_async_shared();
                        void* to = direct ? (void*)(static_cast<__nv_bfloat16*>(a.out) + (size_t)token * a.out_stride + (size_t)head * HD) : (void*)(a.acc + slot * HD);
                        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(smem_u32(room)), "r"(direct ? HD * 2 : HD * 4) : "memory");
                        bulk_commit();
                        bulk_wait<0>();
                    }
                }
            }
        }
    }

    tcgen05_fence_before();
    __syncthreads();
    if (*abort_flag) {                                       // a wait ran out: copies in flight get their time before the block leaves
        for (int i = 0; i < 100; ++i) __nanosleep(10000);
        __syncthreads();
    }
    if (warp == 1) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(COLS) : "memory");
    }
}

// ------------------------------------------------------------------------------------------------ the parts joined
//
// The (token, head) of a row of parts, -1 if it has none: `whole` walks have parts for the tiles that are cut only.
__device__ __forceinline__ int row_of_parts(const Args& a, int row, int n_rows) {
    if (row >= n_rows) return -1;
    if (!a.whole) return row;
    int tile = a.full_tiles + row / WIDE_ROWS, share = a.n_heads / a.n_kv_heads;
    int kv_head = tile % a.n_kv_heads, group = tile / a.n_kv_heads / a.prefix_tiles;
    int at = tile / a.n_kv_heads % a.prefix_tiles * WIDE_ROWS + row % WIDE_ROWS;
    int first = a.cu_seqlens[a.group_first[group]], last = a.cu_seqlens[a.group_first[group + 1]];
    if (at >= (last - first) * share) return -1;
    return (first + at / share) * a.n_heads + kv_head * share + at % share;
}

// WARPS warps a row: each reads all the maxima and sums, a lane a part, and takes every WARPS-th part, several of them in flight; their
// sums are added in order. With one warp that read part after part the join of 34 parts of 512 rows took 25 us, more than the parts.
// CHUNKS: 128 columns of the head each; with two for all sizes the registers let three blocks on an SM, and 2,048 rows of 19 parts took 14 us.
template <typename T, int WARPS, int CHUNKS>
__global__ void __launch_bounds__(256, CHUNKS == 1 ? 5 : 3) prefix_attention_join_kernel(const __grid_constant__ Args a, int n_rows) {
    constexpr int ROWS = 8 / WARPS, AHEAD = 4;
    __shared__ float4 shared_value[8][CHUNKS * 32];
    griddep_launch();
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = warp % WARPS;
    const int row = blockIdx.x * ROWS + warp / WARPS;
    const int D = a.head_dim, slots = a.slots, width = (D + 3) / 4;
    const int of = row_of_parts(a, row, n_rows);
    const bool valid = of >= 0, vectors = D % 4 == 0;
    float4 value[CHUNKS];
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) value[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (valid) {
        const float* acc = behind_wait(a.acc) + (size_t)row * slots * D;
        const float2* stats = reinterpret_cast<const float2*>(behind_wait(a.stats)) + (size_t)row * slots;
        static_assert(MAX_SLOTS <= 128, "four parts a lane");
        float2 part[4];
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            part[k] = lane + 32 * k < slots ? stats[lane + 32 * k] : make_float2(-INFINITY, 0.f);
            m = fmaxf(m, part[k].x);
        }
        m = warp_max(m);
        const float against = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            // (a part without keys has written no values; a sum that is not a number stays one)
            part[k].x = part[k].y != 0.f ? exp2f(part[k].x - against) : 0.f;
            sum += part[k].x * part[k].y;
        }
        sum = warp_sum(sum);
        auto at = [&](int s, int c) {
            int col = (c * 32 + lane) * 4;
            const float* from = acc + (size_t)s * D + col;
            if (vectors) return col < D ? *reinterpret_cast<const float4*>(from) : make_float4(0.f, 0.f, 0.f, 0.f);
            return make_float4(col < D ? from[0] : 0.f, col + 1 < D ? from[1] : 0.f, col + 2 < D ? from[2] : 0.f, col + 3 < D ? from[3] : 0.f);
        };
        for (int s0 = mine; s0 < slots; s0 += WARPS * AHEAD) {
            float weight[AHEAD];
            float4 x[AHEAD][CHUNKS];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                int s = s0 + j * WARPS, k = s >> 5;
                float w = k == 0 ? part[0].x : k == 1 ? part[1].x : k == 2 ? part[2].x : part[3].x;
                weight[j] = __shfl_sync(0xffffffffu, w, s & 31);
                if (s >= slots) weight[j] = 0.f;
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c)
                    x[j][c] = weight[j] != 0.f && c * 128 < D ? at(s, c) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    value[c].x = fmaf(weight[j], x[j][c].x, value[c].x);
                    value[c].y = fmaf(weight[j], x[j][c].y, value[c].y);
                    value[c].z = fmaf(weight[j], x[j][c].z, value[c].z);
                    value[c].w = fmaf(weight[j], x[j][c].w, value[c].w);
                }
        }
    }
    if (WARPS > 1) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            if (c * 32 + lane < width) shared_value[warp][c * 32 + lane] = value[c];
        __syncthreads();
        if (mine) return;
#pragma unroll
        for (int k = 1; k < WARPS; ++k)
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
                if (c * 32 + lane < width) {
                    float4 x = shared_value[warp + k][c * 32 + lane];
                    value[c].x += x.x;
                    value[c].y += x.y;
                    value[c].z += x.z;
                    value[c].w += x.w;
                }
    }
    if (!valid) return;
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    T* out = static_cast<T*>(a.out) + (size_t)(of / a.n_heads) * a.out_stride + (size_t)(of % a.n_heads) * D;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        int col = (c * 32 + lane) * 4;
        float x[4] = {value[c].x * inv, value[c].y * inv, value[c].z * inv, value[c].w * inv};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (col + k < D) out[col + k] = from_float<T>(x[k]);
    }
}

// ------------------------------------------------------------------------------------------------ the call

enum Kernel { CUDA_CORES, FEW, TILE, WIDE };

struct Plan {
    Kernel kernel;                   // of the shared pages
    bool whole;                      // a group's tiles walk the shared and the own pages, nothing is left for own parts
    bool alone;                      // a sequence's own part has the shared pages too
    bool longest_first;              // own slices of long sequences first
    int prefix_tiles, prefix_splits, own_tiles, own_splits, slots, full_tiles;
    long long prefix_blocks, own_blocks;      // one launch, or two with TILE and WIDE
    long long even_blocks;           // > 0: the blocks that deal out unequal groups' pages
    long long part_rows;             // rows that are joined from parts
};

struct Sizes {
    int n_tokens, n_seqs, n_groups, n_heads, n_kv_heads, head_dim, max_new, max_group, max_shared, max_own;
    bool tc;                         // the tensor-core kernels can take the call
};

// Which kernel, and into how many parts the shared and the own pages are cut: as many pages a block as make all blocks come to about the blocks
// that the SMs hold at once, two pages at least.
Plan plan_for(const Sizes& z) {
    Plan p;
    int share = z.n_heads / z.n_kv_heads;
    int shared = z.max_shared > 0 ? bucket(z.max_shared) : 0, own = bucket(ceil_div(z.max_own > 0 ? z.max_own : 1, LLMB_PAGE));
    // sequences that bring few rows each would leave a tile of a group to walk many sequences' pages for a few of its rows
    p.whole = z.tc && (long long)z.max_new * share > FEW_ROWS;
    long long group_rows = shared > 0 ? (long long)z.max_group * share : 0;
    p.alone = reads_alone((long long)z.n_seqs * z.n_kv_heads, shared, group_rows, z.tc, p.whole);
    if (p.alone) {
        own = bucket(own + shared);
        shared = 0;
        group_rows = 0;
    }
    p.kernel = !z.tc ? CUDA_CORES : p.whole || group_rows > TC_ROWS ? WIDE : group_rows > FEW_ROWS ? TILE : FEW;
    int rows = p.kernel == WIDE ? WIDE_ROWS : z.tc ? TC_ROWS : SIMT_ROWS;
    p.prefix_tiles = shared > 0 || p.whole ? ceil_div((long long)z.max_group * share, rows) : 0;
    p.own_tiles = p.whole ? 0 : ceil_div((long long)z.max_new * share, z.tc ? TC_ROWS : SIMT_ROWS);
    p.full_tiles = 0;
    p.even_blocks = 0;
    long long wide_blocks = 0;
    long long prefix = (long long)z.n_groups * p.prefix_tiles * z.n_kv_heads, owns = (long long)z.n_seqs * p.own_tiles * z.n_kv_heads;
    int walk = shared + (p.whole ? own : 0);
    // Several groups: their pages are dealt out on the device, where their lengths are known. Below is then the most that a group is cut into, and the blocks
    // for it: the wide kernel's in one round, the other's as many again as there are groups.
    const bool even = z.tc && !p.whole && z.n_groups > 1 && shared > 0 && z.n_seqs <= STAGED_SEQS;
    if (p.kernel == WIDE) {
        // whole rounds of tiles as they are, the tiles of the last round cut so that they fill one, into four pages at least
        p.full_tiles = p.whole ? (int)(prefix / SMS * SMS) : 0;
        const long long rest = prefix - p.full_tiles;
        p.prefix_splits = wide_pieces(rest, walk, z.head_dim);
        wide_blocks = p.full_tiles + rest * p.prefix_splits;
        p.own_splits = p.own_tiles > 0 ? ceil_div(own, 32) : 0;      // own pages: a launch of their own, 32 pages a block at most
        if (even) {
            p.prefix_splits = ceil_div(SMS, z.n_kv_heads);
            wide_blocks = prefix > SMS ? prefix : SMS;
            p.even_blocks = wide_blocks;
        }
    } else {
        // (on the CUDA cores two blocks fit, and short blocks in a round and a half beat longer ones in one: eight sequences of 4,096 positions 24.9 us for 30.4)
        long long wave = (long long)SMS * (z.tc ? 2 : z.head_dim <= 64 ? 3 : z.head_dim <= 128 ? 2 : 1);
        long long per = (prefix * walk + owns * own + wave - 1) / wave;
        if (per < 2) per = 2;
        p.prefix_splits = p.prefix_tiles > 0 ? ceil_div(walk, per) : 0;
        // own pages beside the tile kernel: a launch of their own, cut only where they are long (16 sequences behind 8,192 positions 17.8 us, with
        // two blocks for one to four own pages 21.9)
        p.own_splits = p.own_tiles == 0 ? 0 : ceil_div(own, p.kernel == TILE ? 32 : per);
        if (even) {
            p.prefix_splits = ceil_div(2 * SMS, z.n_kv_heads);
            if (p.prefix_splits > ceil_div(shared, 2)) p.prefix_splits = ceil_div(shared, 2);
            p.even_blocks = prefix + 2 * SMS;
        }
    }
    if (p.prefix_splits > MAX_SPLITS) p.prefix_splits = MAX_SPLITS;
    if (p.own_splits > MAX_SPLITS) p.own_splits = MAX_SPLITS;
    p.prefix_blocks = p.kernel == WIDE ? wide_blocks : even ? p.even_blocks : prefix * p.prefix_splits;
    p.own_blocks = owns * p.own_splits;
    // Own slices of a launch of their own that make one to two rounds of blocks: the longest first. 64 sequences (8 key heads of 128) with 64 to 1,024
    // positions behind 64 pages 52.4 -> 48.3 us, 40 with up to 2,000 50.0 -> 43.7, 64 of equal length 44.6 -> 46.1 (each block has to find the order). In
    // three rounds the order costs more than it saves (100 sequences 71.4 -> 72.9), beside the shared pages' slices of one launch too.
    p.longest_first = z.tc && !p.whole && (p.kernel != FEW || shared == 0) && own >= 8 && z.n_seqs <= ORDERED_SEQS && p.own_blocks > 2 * SMS && p.own_blocks <= 4 * SMS;
    p.slots = p.prefix_splits + p.own_splits;
    p.part_rows = p.slots == 1 ? 0 : p.whole ? (prefix - p.full_tiles) * WIDE_ROWS : (long long)z.n_tokens * z.n_heads;
    return p;
}

// of the parts' weighted values (their maxima and sums start on 16 bytes behind them), and of both
long long value_floats(long long parts, int head_dim) { return (parts * head_dim + 3) / 4 * 4; }
long long scratch_floats_of(long long parts, int head_dim) { return value_floats(parts, head_dim) + 2 * parts; }

template <typename T, int DMAX>
int launch_simt(const Args& a, unsigned blocks, cudaStream_t stream) {
    constexpr size_t smem = simt_floats<DMAX>() * sizeof(float);
    static bool configured = false;
    if (!configured) {
        LLMB_CUDA(cudaFuncSetAttribute(prefix_attention_simt_kernel<T, DMAX>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        configured = true;
    }
    llmb::launch(prefix_attention_simt_kernel<T, DMAX>, dim3(blocks), SIMT_THREADS, smem, stream, true, a);
    return check_launch("prefix_attention_simt");
}

template <int HD>
int launch_tc(const Args& a, const Plan& p, int n_pages, cudaStream_t stream) {
    // (more than a third of an SM's shared memory: no third block lands there and waits for tensor memory)
    constexpr size_t tiles = 1024 + Ring<HD>::BYTES + 16 * 8;
    static_assert(2 * (tiles + sizeof(Staged) + 1024) <= 227 * 1024 && 2 * Ring<HD>::STAGES <= 14, "two blocks an SM");
    // (more than half of an SM's shared memory for the smaller head size too: tensor memory has room for one block)
    constexpr size_t wide_need = 1024 + (HD / 64) * (2 * Q_PIECE + 4 * PAIR_PIECE) + 19 * 8, wide = wide_need < 120 * 1024 ? 120 * 1024 : wide_need;
    static_assert(wide + sizeof(Staged) + 1024 <= 227 * 1024, "one block an SM");
    static bool configured = false;
    if (!configured) {
        LLMB_CUDA(cudaFuncSetAttribute(prefix_attention_few_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tiles));
        LLMB_CUDA(cudaFuncSetAttribute(prefix_attention_tile_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tiles));
        LLMB_CUDA(cudaFuncSetAttribute(prefix_attention_wide_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)wide));
        cudaFuncAttributes built;                // (its softmax warps would wait for registers that are not there)
        LLMB_CUDA(cudaFuncGetAttributes(&built, prefix_attention_wide_kernel<HD>));
        LLMB_REQUIRE(built.numRegs >= WIDE_REGS_LAUNCHED, "prefix_attention: built with %d registers a thread", built.numRegs);
        configured = true;
    }
    CUtensorMap map_k, map_v;
    long long cache_rows = (long long)n_pages * a.n_kv_heads * LLMB_PAGE;
    int code = make_map_2d(&map_k, a.k_cache, cache_rows, HD, HD, 64, LLMB_PAGE);
    if (!code) code = make_map_2d(&map_v, a.v_cache, cache_rows, HD, HD, 64, LLMB_PAGE);
    if (code) return code;
    static int* status_dev = nullptr;
    if (!status_dev && status_word()) LLMB_CUDA(cudaHostGetDevicePointer((void**)&status_dev, status_word(), 0));
    const unsigned prefix = (unsigned)p.prefix_blocks, own = (unsigned)p.own_blocks;
    if (p.kernel == FEW) {
        llmb::launch(prefix_attention_few_kernel<HD>, dim3(prefix + own), FEW_THREADS, tiles, stream, true, map_k, map_v, a, status_dev);
        return check_launch("prefix_attention_few");
    }
    if (p.kernel == WIDE) llmb::launch(prefix_attention_wide_kernel<HD>, dim3(prefix), WIDE_THREADS, wide, stream, true, map_k, map_v, a, status_dev);
    else llmb::launch(prefix_attention_tile_kernel<HD>, dim3(prefix), TILE_THREADS, tiles, stream, true, map_k, map_v, a, status_dev);
    if ((code = check_launch("prefix_attention_shared")) || own == 0) return code;
    Args behind = a;                          // the own parts, their slots behind those of the shared ones
    behind.prefix_tiles = 0;
    behind.behind = pdl_enabled() ? 1 : 0;
    llmb::launch(prefix_attention_few_kernel<HD>, dim3(own), FEW_THREADS, tiles, stream, true, map_k, map_v, behind, status_dev);
    return check_launch("prefix_attention_few");
}

// a warp for four parts, as many as fit
template <typename T, int CHUNKS>
void launch_join(const Args& a, int rows, cudaStream_t stream) {
    if (a.slots <= 4) llmb::launch(prefix_attention_join_kernel<T, 1, CHUNKS>, dim3((rows + 7) / 8), 256, 0, stream, true, a, rows);
    else if (a.slots <= 8) llmb::launch(prefix_attention_join_kernel<T, 2, CHUNKS>, dim3((rows + 3) / 4), 256, 0, stream, true, a, rows);
    else if (a.slots <= 16) llmb::launch(prefix_attention_join_kernel<T, 4, CHUNKS>, dim3((rows + 1) / 2), 256, 0, stream, true, a, rows);
    else llmb::launch(prefix_attention_join_kernel<T, 8, CHUNKS>, dim3(rows), 256, 0, stream, true, a, rows);
}

int run(const Args& a, const Plan& p, int dtype, int n_pages, cudaStream_t stream) {
    const long long blocks = p.prefix_blocks + p.own_blocks;
    LLMB_REQUIRE(blocks < (1ll << 31), "prefix_attention: too many blocks");
    const bool f32 = dtype == LLMB_DTYPE_F32;
    int code;
    if (p.kernel != CUDA_CORES) code = a.head_dim == 64 ? launch_tc<64>(a, p, n_pages, stream) : launch_tc<128>(a, p, n_pages, stream);
    else if (a.head_dim <= 64) code = f32 ? launch_simt<float, 64>(a, (unsigned)blocks, stream) : launch_simt<__nv_bfloat16, 64>(a, (unsigned)blocks, stream);
    else if (a.head_dim <= 128) code = f32 ? launch_simt<float, 128>(a, (unsigned)blocks, stream) : launch_simt<__nv_bfloat16, 128>(a, (unsigned)blocks, stream);
    else code = f32 ? launch_simt<float, 256>(a, (unsigned)blocks, stream) : launch_simt<__nv_bfloat16, 256>(a, (unsigned)blocks, stream);
    if (code || a.slots == 1) return code;
    const bool narrow = a.head_dim <= 128;
    if (f32) narrow ? launch_join<float, 1>(a, (int)p.part_rows, stream) : launch_join<float, 2>(a, (int)p.part_rows, stream);
    else narrow ? launch_join<__nv_bfloat16, 1>(a, (int)p.part_rows, stream) : launch_join<__nv_bfloat16, 2>(a, (int)p.part_rows, stream);
    return check_launch("prefix_attention_join");
}

}  // namespace

LLMB_EXPORT int llmb_prefix_attention_status() {
    int* s = status_word();
    if (!s) return -1;
    int v = *s;
    *s = 0;
    return v;
}

// The sizes of a call, one integer each.
struct llmb_prefix_sizes {
    int q_stride, n_pages, table_stride, out_stride;         // elements between rows, pages of the caches
    int dtype, n_tokens, n_seqs, n_groups, n_heads, n_kv_heads, head_dim;
    int max_new, max_group, max_shared, max_own;             // upper bounds (ops.prefix_attention)
    int tc;                                                  // whether the tensor-core kernels take the call (refused where they cannot), 0: the CUDA cores
};

namespace {
Sizes sizes_of(const llmb_prefix_sizes& z) {
    return Sizes{z.n_tokens, z.n_seqs, z.n_groups, z.n_heads, z.n_kv_heads, z.head_dim, z.max_new, z.max_group, z.max_shared, z.max_own, z.tc != 0};
}
}  // namespace

// Floats of scratch that a call of these sizes needs, and the number of its launches in *kernels.
LLMB_EXPORT long long llmb_prefix_attention_scratch_floats(const llmb_prefix_sizes* z, int* kernels) {
    *kernels = 1;
    if (z->n_tokens <= 0 || z->n_seqs <= 0 || z->n_groups <= 0 || z->n_kv_heads <= 0 || z->n_heads < z->n_kv_heads) return 0;
    Plan p = plan_for(sizes_of(*z));
    if (p.slots > 1) ++*kernels;
    if ((p.kernel == TILE || p.kernel == WIDE) && p.own_blocks > 0) ++*kernels;
    return scratch_floats_of(p.part_rows * p.slots, z->head_dim);
}

LLMB_EXPORT int llmb_prefix_attention(const void* q, const void* k_cache, const void* v_cache, const int* block_table, const int* seq_lens,
                                      const int* cu_seqlens, const int* group_first, const int* group_pages, void* out, float* scratch,
                                      long long scratch_floats, float scale, const llmb_prefix_sizes* sizes, cudaStream_t stream) {
    const llmb_prefix_sizes& z = *sizes;
    if (z.n_tokens == 0 || z.n_seqs == 0) return LLMB_OK;
    LLMB_REQUIRE(z.dtype == LLMB_DTYPE_F32 || z.dtype == LLMB_DTYPE_BF16, "prefix_attention: float32 and bfloat16 are built");
    LLMB_REQUIRE(z.n_tokens > 0 && z.n_seqs > 0 && z.n_groups > 0 && z.n_groups <= z.n_seqs, "prefix_attention: %d tokens of %d sequences in %d groups",
                 z.n_tokens, z.n_seqs, z.n_groups);
    LLMB_REQUIRE(z.n_kv_heads > 0 && z.n_heads > 0 && z.n_heads % z.n_kv_heads == 0, "prefix_attention: %d heads are no multiple of %d kv heads",
                 z.n_heads, z.n_kv_heads);
    LLMB_REQUIRE(z.head_dim > 0 && z.head_dim <= LLMB_MAX_HEAD_DIM, "prefix_attention: head_dim %d (served: up to %d)", z.head_dim, LLMB_MAX_HEAD_DIM);
    LLMB_REQUIRE(z.max_new > 0 && z.max_group >= z.max_new && z.max_shared >= 0 && z.max_own >= 0, "prefix_attention: bad sizes");
    LLMB_REQUIRE((long long)z.n_tokens * z.n_heads < (1ll << 31), "prefix_attention: %d tokens of %d heads", z.n_tokens, z.n_heads);
    auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    LLMB_REQUIRE(!z.tc || (z.dtype == LLMB_DTYPE_BF16 && (z.head_dim == 64 || z.head_dim == 128) && scale > 0.f && z.q_stride % 8 == 0 && z.out_stride % 8 == 0 &&
                           aligned(q) && aligned(out) && aligned(k_cache) && aligned(v_cache)),
                 "prefix_attention: the tensor-core kernels do not take these operands");
    LLMB_REQUIRE(z.n_pages > 0 && (long long)z.n_pages * z.n_kv_heads * LLMB_PAGE < (1ll << 31), "prefix_attention: %d pages", z.n_pages);
    Plan p = plan_for(sizes_of(z));
    const long long parts = p.part_rows * p.slots;
    LLMB_REQUIRE(p.part_rows < (1ll << 31), "prefix_attention: %lld rows of parts", p.part_rows);
    LLMB_REQUIRE(parts == 0 || (scratch != nullptr && aligned(scratch) && scratch_floats >= scratch_floats_of(parts, z.head_dim)),
                 "prefix_attention: scratch too small");
    bool vectors = (z.head_dim * (z.dtype == LLMB_DTYPE_F32 ? 4 : 2)) % 16 == 0 && aligned(k_cache) && aligned(v_cache);
    Args a{q, k_cache, v_cache, block_table, seq_lens, cu_seqlens, group_first, group_pages, out, scratch, scratch + value_floats(parts, z.head_dim),
           z.q_stride, z.out_stride, z.table_stride, z.n_seqs, z.n_groups, z.n_heads, z.n_kv_heads, z.head_dim, scale * LOG2E,
           p.prefix_tiles, p.prefix_splits, p.own_tiles, p.own_splits, p.slots, vectors ? 1 : 0, p.full_tiles,
           (int)p.even_blocks, 0, p.longest_first ? 1 : 0, nullptr, p.alone ? 1 : 0, p.whole ? 1 : 0};
    return run(a, p, z.dtype, z.n_pages, stream);
}

// the packed doors of the launching entry points (common.cuh)
LLMB_PACKED(llmb_prefix_attention)
