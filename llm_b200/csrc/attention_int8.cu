// Causal grouped-query attention over a paged cache that is held in 8 bits (int8_pages.cuh).
//
//   out[t, a] = sum_j p_j v_j,  p = softmax_j(scale * q[t, a] . k_j),  j <= position of t and j > position - window (window > 0),
//   keys of head a * kv_heads / heads, k_j and v_j a whole number times the scale of the position's block
//
// A row is (token, query head of the key head): row r of a sequence is its token r / share, head r % share, with share = heads / kv_heads, so that
// one pass over a key head serves all query heads that share it. A block has a tile of rows and a slice of the pages that those rows see; each slice
// leaves, per row, (weighted values, maximum, sum), which the last kernel joins with out = sum_i acc_i e^(m_i - m) / sum_i l_i e^(m_i - m) in the order
// of the slices.
//
// Lengths, tables and the order of sequences are read from device arrays; the sizes of the launch are upper bounds. A key that a row does not see has
// no weight whatever is stored there: whole numbers are finite, and a block whose scale is no number counts with the scores of the keys that
// are seen (their weights become no number), never in the products.
#include "int8_pages.cuh"
#include "mma.cuh"
#include "tc.cuh"

using namespace llmb;
using namespace llmb::tc;

LLMB_DEFINE_LAST_ERROR(llmb_attention_int8)

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int SMS = 148;
constexpr int MAX_SPLITS = 64;

struct Args {
    const void* q;
    const signed char* keys;         // [pages, n_kv_heads, 64, head_dim]
    const float* key_scales;         // [pages, n_kv_heads, 64 >> block_shift]
    const signed char* values;
    const float* value_scales;
    const int* block_table;          // [n_seqs, table_stride]
    const int* seq_lens;             // [n_seqs] with the new tokens
    const int* cu_seqlens;           // [n_seqs + 1]
    const int* seq_order;            // [n_seqs] longest first, or none
    void* out;
    float* acc;                      // [n_tokens * n_heads, slots, head_dim]
    float* stats;                    // [n_tokens * n_heads, slots, 2]: maximum in base-2 units, sum
    int q_stride, out_stride, table_stride, ring_pages, n_pages, n_tokens, n_seqs, n_heads, n_kv_heads, head_dim, block_shift, window;
    float scale_log2;
    int max_new, tiles, slots;
    int few_tokens;                  // sequences that bring at most so many tokens are the kernel's for few rows (0: it is not launched)
    int deal_blocks, deal_least;     // its blocks that all pages are dealt out to, in ranges of so many pages at least; 0: a block a (sequence, key head)
    int wide_blocks, wide_least;     // the same of the kernel for many rows, in steps; 0: a block a tile
    float* wide_acc;                 // parts of that kernel's blocks: [blocks, 2, 256, head_dim], and their maxima and sums
    float* wide_stats;
    int2* few_blocks_of;             // [n_seqs, n_kv_heads] which blocks have parts of a pair, [n_seqs, n_kv_heads, tiles] of a tile
    int2* wide_blocks_of;
    int* arrived;                    // [n_seqs, n_kv_heads] zeros: how many of a pair's parts are there, where its last block joins them (null: a launch does)
};

// What a kernel reports (no wait has these codes): a step that brings more tokens than max_new says; a place outside of what the call was given, which is
// not read: a page, a token or a sequence that there is not; a scale of what is seen that is no power of two; scores beyond LARGEST_SCORE.
constexpr int BEYOND_BOUNDS = 50, OUT_OF_RANGE = 51, NOT_A_POWER = 52, LARGE_SCORES = 53;
__device__ __forceinline__ void report(int* status, int code) {
    if (status) atomicCAS(status, 0, code);
}

// A block's share of the work: rows of a sequence against a slice of its pages.
struct Item {
    int kv_head, seq, slot;
    int first_token, row0, n_rows;   // the sequence's first token; rows row0 .. row0 + n_rows - 1 of the sequence
    int first_pos;                   // position of the sequence's first new token
    int page_begin, page_end;        // places in the table, before the ring
};

// the first key that a position sees
__device__ __forceinline__ int first_seen(const Args& a, int position) { return a.window > 0 ? max(position - a.window + 1, 0) : 0; }
// How many pages the new tokens of a sequence see: more than its ring has are not there any more (one would be read in another's place).
__device__ __forceinline__ int pages_seen(const Args& a, int first_pos, int n_new) {
    return (first_pos + n_new - 1) / LLMB_PAGE + 1 - first_seen(a, first_pos) / LLMB_PAGE;
}

// false where nothing is left for the block
__device__ __forceinline__ bool item_of(const Args& a, int x, int slot, int tile_rows, Item& w, int* status) {
    w.kv_head = x % a.n_kv_heads;
    x /= a.n_kv_heads;
    const int back = x % a.tiles, share = a.n_heads / a.n_kv_heads;
    x /= a.tiles;
    w.seq = a.seq_order ? a.seq_order[x] : x;
    w.slot = slot;
    if ((unsigned)w.seq >= (unsigned)a.n_seqs) {
        if (threadIdx.x == 0) report(status, OUT_OF_RANGE);
        return false;
    }
    w.first_token = a.cu_seqlens[w.seq];
    const int end_token = a.cu_seqlens[w.seq + 1];
    int n_new = end_token - w.first_token;
    w.first_pos = a.seq_lens[w.seq] - n_new;
    if (w.first_token < 0 || end_token > a.n_tokens || (n_new > 0 && (w.first_pos < 0 || pages_seen(a, w.first_pos, n_new) > a.ring_pages))) {
        if (threadIdx.x == 0) report(status, OUT_OF_RANGE);
        return false;
    }
    if (n_new > a.max_new) {                                  // rows that no block has
        if (threadIdx.x == 0) report(status, BEYOND_BOUNDS);
        n_new = a.max_new;
    }
    const int tiles = (n_new * share + tile_rows - 1) / tile_rows;
    if (back >= tiles) return false;
    const int tile = tiles - 1 - back;                        // those that see most start first
    w.row0 = tile * tile_rows;
    w.n_rows = min(tile_rows, n_new * share - w.row0);
    const int first = w.first_pos + w.row0 / share, last = w.first_pos + (w.row0 + w.n_rows - 1) / share;
    const int begin = a.window > 0 ? max(first - a.window + 1, 0) / LLMB_PAGE : 0, end = last / LLMB_PAGE + 1;
    const int per = (end - begin + a.slots - 1) / a.slots;
    w.page_begin = begin + min(slot * per, end - begin);
    w.page_end = min(w.page_begin + per, end);
    return true;
}
__device__ __forceinline__ int token_of(const Item& w, int r, int share) { return w.first_token + (w.row0 + r) / share; }
__device__ __forceinline__ int head_of(const Item& w, int r, int share) { return w.kv_head * share + (w.row0 + r) % share; }
__device__ __forceinline__ int position_of(const Item& w, int r, int share) { return w.first_pos + (w.row0 + r) / share; }
// the page of a place in the table; one that there is not is reported, and page 0 read in its place
__device__ __forceinline__ int page_at(const Args& a, const int* pages, int logical, int* status) {
    if (logical >= a.ring_pages) logical %= a.ring_pages;      // (a division only where the ring has been gone round)
    const int page = pages[logical];
    if ((unsigned)page < (unsigned)a.n_pages) return page;
    report(status, OUT_OF_RANGE);
    return 0;
}

// ------------------------------------------------------------------------------------------------ any type, any head size
//
// 32-bit arithmetic on the CUDA cores: the path of 32-bit queries, and of the head sizes that the tensor-core kernels are not built for. A block holds
// 32 rows and walks its pages one by one: 64 keys and values in shared memory as 32-bit values, four rows a warp. A lane forms their scores with
// keys `lane` and `lane + 32`, shares the maxima with the others, and adds the weighted values of its columns, two multiply-adds to an instruction.
// Rows of a key or value are 4 words longer than the head, so that the eight rows that are read at a time lie in different banks. A page's 8-bit
// rows are one piece; they are fetched to registers a step ahead and widened on their way to shared memory.

constexpr int SIMT_ROWS = 32, SIMT_THREADS = 256, RT = SIMT_ROWS / (SIMT_THREADS / 32);     // RT: rows of a warp

// two 32-bit values to an instruction
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) { return pair_of(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float half_of(uint64_t v, int which) { return __uint_as_float((uint32_t)(which ? v >> 32 : v)); }
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
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }

template <int DMAX>
constexpr int simt_floats() { return (SIMT_ROWS + 2 * LLMB_PAGE) * (DMAX + 4) + SIMT_ROWS * LLMB_PAGE; }

template <typename T, int DMAX>
__global__ void __launch_bounds__(SIMT_THREADS) attention_int8_simt_kernel(const __grid_constant__ Args a, int* status) {
    constexpr int LD = DMAX + 4, W = DMAX == 64 ? 2 : 4, COLS = DMAX / (32 * W);      // a lane's columns: COLS times W that adjoin
    constexpr int FETCH = DMAX * LLMB_PAGE / (16 * SIMT_THREADS);                    // 16-byte pieces of a page's rows, of a thread
    extern __shared__ __align__(16) float smem[];
    float* qs = smem;                              // [32][LD], scaled
    float* ks = qs + SIMT_ROWS * LD;               // [64][LD]
    float* vs = ks + LLMB_PAGE * LD;               // [64][LD]
    float* ps = vs + LLMB_PAGE * LD;               // [warp][64 keys][4 rows]

    griddep_launch();
    const int tid = threadIdx.x, ty = tid >> 5, tx = tid & 31;
    for (int i = tid; i < 2 * LLMB_PAGE * LD; i += SIMT_THREADS) ks[i] = 0.f;        // columns behind the head's last
    griddep_wait();
    Item w;
    if (!item_of(a, blockIdx.x, blockIdx.y, SIMT_ROWS, w, status)) return;
    const int D = a.head_dim, share = a.n_heads / a.n_kv_heads;
    const T* q = behind_wait(static_cast<const T*>(a.q));
    const int* pages = a.block_table + (size_t)w.seq * a.table_stride;
    const int scales_per_page = LLMB_PAGE >> a.block_shift;

    uint4 fetched[FETCH];
    auto fetch = [&](const signed char* cache, int page) {
        const uint4* from = reinterpret_cast<const uint4*>(cache + ((size_t)page * a.n_kv_heads + w.kv_head) * LLMB_PAGE * D);
#pragma unroll
        for (int j = 0; j < FETCH; ++j)
            if (tid + j * SIMT_THREADS < 4 * D) fetched[j] = from[tid + j * SIMT_THREADS];
    };
    auto widen = [&](float* to, const float* scales) {         // scales of the page
#pragma unroll
        for (int j = 0; j < FETCH; ++j) {
            const int piece = tid + j * SIMT_THREADS;
            if (piece >= 4 * D) break;
            int row = piece * 16 / D, col = piece * 16 - row * D;
            float s = scales[row >> a.block_shift];
            if (!is_number(s)) s = 0.f;
            const signed char* x = reinterpret_cast<const signed char*>(&fetched[j]);
            if (D % 16 == 0) {
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4*>(to + row * LD + col + e) = make_float4(x[e] * s, x[e + 1] * s, x[e + 2] * s, x[e + 3] * s);
            } else {
#pragma unroll 1
                for (int e = 0; e < 16; ++e) {
                    to[row * LD + col] = x[e] * s;
                    if (++col == D) {
                        col = 0;
                        ++row;
                        s = row < LLMB_PAGE ? scales[row >> a.block_shift] : 0.f;
                        if (!is_number(s)) s = 0.f;
                    }
                }
            }
        }
    };

#pragma unroll 4
    for (int r = ty; r < SIMT_ROWS; r += SIMT_THREADS / 32) {          // a warp a row
        const bool valid = r < w.n_rows;
        const T* from = q + (size_t)token_of(w, valid ? r : 0, share) * a.q_stride + (size_t)head_of(w, valid ? r : 0, share) * D;
#pragma unroll
        for (int d = tx; d < DMAX; d += 32) qs[r * LD + d] = valid && d < D ? to_float(from[d]) * a.scale_log2 : 0.f;
    }
    float m[RT], l[RT];
    uint64_t o[RT / 2][COLS * W];                  // of rows 2 i and 2 i + 1
    float4* weights = reinterpret_cast<float4*>(ps) + ty * LLMB_PAGE;
    int pos[RT], seen[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
        pos[i] = ty * RT + i < w.n_rows ? position_of(w, ty * RT + i, share) : -1;
        seen[i] = first_seen(a, pos[i]);
    }
#pragma unroll
    for (int i = 0; i < RT / 2; ++i)
#pragma unroll
        for (int c = 0; c < COLS * W; ++c) o[i][c] = 0;
    const bool idle = ty * RT >= w.n_rows;                     // a warp without rows
    const int last = position_of(w, w.n_rows - 1, share), low = first_seen(a, position_of(w, 0, share));      // what a row of the tile sees at all
    if (w.page_begin < w.page_end) fetch(a.keys, page_at(a, pages, w.page_begin, status));
    for (int logical = w.page_begin; logical < w.page_end; ++logical) {
        const int key0 = logical * LLMB_PAGE, page = page_at(a, pages, logical, status);
        const size_t at = ((size_t)page * a.n_kv_heads + w.kv_head) * scales_per_page;
        const float* k_scales = a.key_scales + at;
        const float* v_scales = a.value_scales + at;
        widen(ks, k_scales);
        fetch(a.values, page);
        __syncthreads();                           // the keys are there, everyone is done with the values before
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
            float weight[2][RT], alpha[RT], bad[2];          // bad: 0, or no number where a scale is none
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int b = (tx + 32 * j) >> a.block_shift;
                const float sk = k_scales[b], sv = v_scales[b];
                bad[j] = is_number(sk) && is_number(sv) ? 0.f : __uint_as_float(0x7fffffffu);
                if (bad[j] == 0.f && key0 + tx + 32 * j <= last && ((__float_as_uint(sk) | __float_as_uint(sv)) & 0x807fffffu) &&
                    key0 + tx + 32 * j >= low) report(status, NOT_A_POWER);
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                float s[2], top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int key = key0 + tx + 32 * j;
                    s[j] = key > pos[i] || key < seen[i] ? -INFINITY : half_of(dot[i][j], 0) + half_of(dot[i][j], 1) + bad[j];
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
        widen(vs, v_scales);
        __syncthreads();                           // the values are there, everyone is done with the keys
        if (logical + 1 < w.page_end) fetch(a.keys, page_at(a, pages, logical + 1, status));
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
    if (idle) return;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        l[i] = warp_sum(l[i]);
        const int r = ty * RT + i;
        if (r >= w.n_rows) continue;
        const int token = token_of(w, r, share), head = head_of(w, r, share);
        if (a.slots == 1) {
            const float inv = l[i] != 0.f ? 1.f / l[i] : 0.f;
            T* to = static_cast<T*>(a.out) + (size_t)token * a.out_stride + (size_t)head * D;
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
                for (int x = 0; x < W; ++x)
                    if ((c * 32 + tx) * W + x < D) to[(c * 32 + tx) * W + x] = from_float<T>(half_of(o[i / 2][c * W + x], i & 1) * inv);
        } else {
            const size_t slot = ((size_t)token * a.n_heads + head) * a.slots + w.slot;
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
                for (int x = 0; x < W; ++x)
                    if ((c * 32 + tx) * W + x < D) a.acc[slot * D + (c * 32 + tx) * W + x] = half_of(o[i / 2][c * W + x], i & 1);
            if (tx == 0) *reinterpret_cast<float2*>(a.stats + slot * 2) = make_float2(l[i] != 0.f ? m[i] : -INFINITY, l[i]);
        }
    }
}

// ------------------------------------------------------------------------------------------------ any type, any head size, up to 8 rows
//
// The same arithmetic for what a decode step brings: with 32 rows a block one warp of eight would have all the work. Here each warp walks pages of its
// own. A lane forms the scores of all rows with keys `lane` and `lane + 32`, whose bytes it reads itself and widens to 32 bits in registers; the
// weights, times the values' scales, go through shared memory; then a lane adds the weighted values of its columns. The eight warps' sums meet at
// the end. Eight sequences of 4,096 positions (32 heads over 8 of 64, 32-bit) take 30 us, with 32 rows a block 73. What bounds it is a page's chain: with the
// keys' and values' loads where they are used it was 77; with one block of eight warps an SM and 165 registers a thread 44, with two and 16 values at a
// time 34, four blocks of four warps 31.

constexpr int ROWS_THREADS = 256, ROWS_WARPS = ROWS_THREADS / 32;

// Four bytes as 32-bit values: 0x4b000000 | (b ^ 0x80) is 8388608 + 128 + b.
__device__ __forceinline__ void widen4(uint32_t x, float (&v)[4]) {
    x ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7650 + i)) - 8388736.f;
}
template <int DMAX, int R> constexpr int rows_floats() { return R * DMAX + ROWS_WARPS * (R * DMAX > LLMB_PAGE * R ? R * DMAX : LLMB_PAGE * R) + ROWS_WARPS * R * 2; }

template <typename T, int DMAX, int R>
__global__ void __launch_bounds__(ROWS_THREADS, DMAX == 64 ? 2 : 1) attention_int8_rows_kernel(const __grid_constant__ Args a, int* status) {
    constexpr int W = DMAX / 32;                   // a lane's columns, which adjoin
    extern __shared__ __align__(16) float smem[];
    float* qs = smem;                              // [R][DMAX], scaled; zeros behind the head's last column
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int ROOM = R * DMAX > LLMB_PAGE * R ? R * DMAX : LLMB_PAGE * R;
    float* room = smem + R * DMAX;                 // of each warp: its weights [64][R], at the end its sums [R][DMAX]
    float* weights = room + warp * ROOM;
    float2* stats = reinterpret_cast<float2*>(room + ROWS_WARPS * ROOM);         // [warp][R]
    griddep_launch();
    Item w;
    const bool work = item_of(a, blockIdx.x, blockIdx.y, R, w, status);
    griddep_wait();
    if (!work) return;
    const int D = a.head_dim, share = a.n_heads / a.n_kv_heads;
    const T* q = behind_wait(static_cast<const T*>(a.q));
    const int* pages = a.block_table + (size_t)w.seq * a.table_stride;
    const int scales_per_page = LLMB_PAGE >> a.block_shift;
    for (int i = threadIdx.x; i < R * DMAX; i += ROWS_THREADS) {
        const int r = i / DMAX, d = i - r * DMAX;
        qs[i] = r < w.n_rows && d < D ? to_float(q[(size_t)token_of(w, r, share) * a.q_stride + (size_t)head_of(w, r, share) * D + d]) * a.scale_log2 : 0.f;
    }
    __syncthreads();
    float m[R], l[R], o[R][W];
    int pos[R], seen[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
        pos[r] = r < w.n_rows ? position_of(w, r, share) : -1;
        seen[r] = first_seen(a, pos[r]);
#pragma unroll
        for (int c = 0; c < W; ++c) o[r][c] = 0.f;
    }
    const int last = position_of(w, w.n_rows - 1, share), low = first_seen(a, position_of(w, 0, share));      // what a row sees at all
    // A page's loads are under way before anything is worked out: the keys' bytes of this lane's two (where the head is not too large for the
    // registers), the scales, the first values; then each group of values under the products with the one before.
    constexpr int HALVES = DMAX <= 128 ? 2 : 1, GROUP = 8, WORDS = (W + 3) / 4;
    const bool vectors = D % 16 == 0, all = lane * W + W <= D && D % W == 0;     // a key's bytes can be read 16 at a time, this lane's columns at once
    int next = w.page_begin + warp < w.page_end ? page_at(a, pages, w.page_begin + warp, status) : 0;
    for (int logical = w.page_begin + warp; logical < w.page_end; logical += ROWS_WARPS) {
        const int key0 = logical * LLMB_PAGE, from = max(low - key0, 0), to = min(last + 1 - key0, LLMB_PAGE);      // what of the page a row sees at all
        const size_t at = (size_t)next * a.n_kv_heads + w.kv_head;
        const signed char* keys = a.keys + at * LLMB_PAGE * D;
        const signed char* values = a.values + at * LLMB_PAGE * D + lane * W;
        if (logical + ROWS_WARPS < w.page_end) next = page_at(a, pages, logical + ROWS_WARPS, status);
        uint4 raw[HALVES][DMAX / 16];
        auto fetch_keys = [&](int half, uint4 (&x)[DMAX / 16]) {
            const int k = lane + 32 * half;
            const uint4* row = reinterpret_cast<const uint4*>(keys + (size_t)k * D);
#pragma unroll
            for (int i = 0; i < DMAX / 16; ++i)
                if (vectors && i * 16 < D && k >= from && k < to) x[i] = row[i];
        };
        uint32_t held[2][GROUP][WORDS];
        auto fetch_values = [&](int k0, uint32_t (&x)[GROUP][WORDS]) {
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                const int k = k0 + j;
                const signed char* row = values + (size_t)k * D;
                if (k >= to || lane * W >= D) continue;
                if (!all) {
#pragma unroll
                    for (int c = 0; c < W; ++c) {
                        if (c % 4 == 0) x[j][c / 4] = 0;
                        if (lane * W + c < D) x[j][c / 4] |= (uint32_t)(unsigned char)row[c] << (8 * (c % 4));
                    }
                } else if constexpr (W == 2) {
                    x[j][0] = *reinterpret_cast<const unsigned short*>(row);
                } else {
#pragma unroll
                    for (int c = 0; c < WORDS; ++c) x[j][c] = reinterpret_cast<const uint32_t*>(row)[c];
                }
            }
        };
        float s[2][R], ks[2], vs[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = lane + 32 * half;
            const bool there = k >= from && k < to;
            ks[half] = there ? a.key_scales[at * scales_per_page + (k >> a.block_shift)] : 0.f;
            vs[half] = there ? a.value_scales[at * scales_per_page + (k >> a.block_shift)] : 0.f;
            if (half < HALVES) fetch_keys(half, raw[half]);
        }
        fetch_values(from, held[0]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = lane + 32 * half, key = key0 + k;
            if (half >= HALVES) fetch_keys(half, raw[0]);
            const uint4 (&x)[DMAX / 16] = raw[half < HALVES ? half : 0];
            const bool bad = !is_number(ks[half]) || !is_number(vs[half]);
            if (!bad && ((__float_as_uint(ks[half]) | __float_as_uint(vs[half])) & 0x807fffffu)) report(status, NOT_A_POWER);
            uint64_t dot[R];                       // even and odd columns apart
#pragma unroll
            for (int r = 0; r < R; ++r) dot[r] = 0;
            auto add = [&](uint32_t bytes, int d) {
                float v[4];
                widen4(bytes, v);
                const uint64_t v01 = pair_of(v[0], v[1]), v23 = pair_of(v[2], v[3]);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const ulonglong2 qv = *reinterpret_cast<const ulonglong2*>(qs + r * DMAX + d);
                    dot[r] = fma2(qv.x, v01, fma2(qv.y, v23, dot[r]));
                }
            };
            if (k >= from && k < to) {
                if (vectors) {
#pragma unroll
                    for (int i = 0; i < DMAX / 16; ++i) {
                        if (i * 16 >= D) break;
                        add(x[i].x, i * 16);
                        add(x[i].y, i * 16 + 4);
                        add(x[i].z, i * 16 + 8);
                        add(x[i].w, i * 16 + 12);
                    }
                } else {
                    const signed char* row = keys + (size_t)k * D;
                    for (int d = 0; d < D; d += 4) {             // (heads are even; the last two columns may be none)
                        uint32_t y = *reinterpret_cast<const unsigned short*>(row + d);
                        if (d + 2 < D) y |= (uint32_t)*reinterpret_cast<const unsigned short*>(row + d + 2) << 16;
                        add(y, d);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                s[half][r] = bad ? __uint_as_float(0x7fffffffu) : (half_of(dot[r], 0) + half_of(dot[r], 1)) * ks[half];
                if (key > pos[r] || key < seen[r]) s[half][r] = -INFINITY;
            }
            if (bad) vs[half] = 0.f;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float top = warp_max(fmaxf(s[0][r], s[1][r]));
            const float new_m = fmaxf(m[r], top), against = new_m == -INFINITY ? 0.f : new_m, alpha = exp2f(m[r] - against);
            m[r] = new_m;
            float add = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float p = exp2f(s[half][r] - against);
                add += p;
                weights[(lane + 32 * half) * R + r] = p * vs[half];
            }
            l[r] = l[r] * alpha + add;             // of this lane's keys
#pragma unroll
            for (int c = 0; c < W; ++c) o[r][c] *= alpha;
        }
        __syncwarp();
        auto multiply = [&](int k0, const uint32_t (&x)[GROUP][WORDS]) {
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                if (k0 + j >= to) break;
                float v[WORDS * 4];
#pragma unroll
                for (int c = 0; c < WORDS; ++c) widen4(x[j][c], *reinterpret_cast<float (*)[4]>(v + 4 * c));
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float p = weights[(k0 + j) * R + r];
#pragma unroll
                    for (int c = 0; c < W; ++c) o[r][c] = fmaf(p, v[c], o[r][c]);
                }
            }
        };
        for (int k = from; k < to; k += 2 * GROUP) {
            fetch_values(k + GROUP, held[1]);
            multiply(k, held[0]);
            fetch_values(k + 2 * GROUP, held[0]);
            multiply(k + GROUP, held[1]);
        }
        __syncwarp();                              // the weights are read before the next page's are written
    }
    // the warps' sums in order
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] = warp_sum(l[r]);
        if (lane == 0) stats[warp * R + r] = make_float2(m[r], l[r]);
#pragma unroll
        for (int c = 0; c < W; ++c) room[warp * ROOM + r * DMAX + lane * W + c] = o[r][c];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < w.n_rows * D; i += ROWS_THREADS) {
        const int r = i / D, d = i - r * D;
        float top = -INFINITY, value = 0.f, sum = 0.f;
#pragma unroll
        for (int k = 0; k < ROWS_WARPS; ++k) top = fmaxf(top, stats[k * R + r].x);
        const float against = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int k = 0; k < ROWS_WARPS; ++k) {
            const float2 of = stats[k * R + r];
            const float weight = of.y != 0.f ? exp2f(of.x - against) : 0.f;
            sum += of.y * weight;
            value = fmaf(room[k * ROOM + r * DMAX + d], weight, value);
        }
        const int token = token_of(w, r, share), head = head_of(w, r, share);
        if (a.slots == 1) {
            static_cast<T*>(a.out)[(size_t)token * a.out_stride + (size_t)head * D + d] = from_float<T>(sum != 0.f ? value / sum : 0.f);
        } else {
            const size_t slot = ((size_t)token * a.n_heads + head) * a.slots + w.slot;
            a.acc[slot * D + d] = value;
            if (d == 0) *reinterpret_cast<float2*>(a.stats + slot * 2) = make_float2(sum != 0.f ? top : -INFINITY, sum);
        }
    }
}

// ------------------------------------------------------------------------------------------------ bfloat16, up to 16 rows
//
// What a decode step brings. Reading the cache is the work, and widening it: 16 bits would be twice the bytes, so the whole numbers stay what they are
// until they are in registers. A byte b (two's complement) is exactly the fp16 number 1024 + 128 + b with the bits 0x6400 | (b ^ 0x80), one
// logical operation for two of them; a multiply-add by (s, -1152 s) leaves b s, exact for s a power of two. Products are mma.sync with the cache's
// positions (for the scores) or the head's columns (for the result) on the 16-row side and the queries' rows, 8 or 16, on the other: what is
// widened is multiplied once.
//
//   scores^T [16 positions, rows] = K [16, D] Q^T        result^T [16 columns, rows] += V^T [16, positions] P^T
//
// fp16 holds 2^-24 to 65504. So queries are divided by the power of two that brings their row's largest to 2^14; scales count from the largest of the
// positions that a warp works on (2^5 for that one, so that 29 powers of two fit); and a row keeps, beside the running maximum m of its scores, a
// reference R of score plus exponent of the values' scale, to which its weights w = 2^(score - m) 2^(m + E - R + 14) and its sums refer (what is held is R - m,
// so that large scores take nothing from it). All sums are in 32 bits. What is lost: values below 2^-29, and weights below 2^-38, of the largest that counts there. That is the
// largest of what any of the rows sees, in a unit for values and so far for weights: a loud position that one row is not to see takes from the others
// what is 2^29 below it.
//
// The pages of all (sequence, key head) pairs, one after the other, are dealt out to the blocks that the SMs hold at once in ranges of
// equal length, so a block's range covers the end of one pair, some whole ones, and the beginning of another. Pairs that one block has done as a whole are
// finished there, of the others each block leaves a part. A block has four warps, each with a ring of units of its own, 32 positions or 64 (TMA, rows
// swizzled so that both the reads of keys, four lanes a row, and those of values, eight columns a lane, touch all banks once), which runs on over the
// ends of pairs; warps meet where a pair ends. Of a pair that several blocks have, a launch joins the parts, or the last block to come (plan_for).
//
// 64 sequences of 8,192 positions (32 heads over 8 of 128, 1.08 GB) take 173 us in short bursts, 6.2 TB/s, and 204 in long loops at the power cap: reading
// is the limit, and the energy of some 770 instructions for 8 KB. Eight take 37 us, one 11 on the device: 10 of them are a block's start (lengths, table,
// first pages: dependent reads), its end and the join. Three blocks an SM of 165 registers; with maximum, reference and masks worked out anew for every unit,
// and 32 positions for heads of 64 too, a unit took 1,130 instructions.

constexpr int FEW_THREADS = 128, FEW_WARPS = 4;
constexpr int FEW_ROWS = 16;
constexpr int SCALE_UP = 5, WEIGHT_UP = 14;                    // powers of two that the largest scale and weight are lifted to

template <int HD> constexpr int UNIT = HD == 64 ? 64 : 32;      // positions that a warp works on at a time
template <int HD, int NT> struct Few {
    static constexpr int TILE = UNIT<HD> * HD;                  // bytes of a unit's keys
    static constexpr int STAGES = 2;
    static constexpr int BLOCKS = NT == 1 ? 3 : 2;              // of an SM
    static constexpr int LD = HD + 4;
    static constexpr int RING = FEW_WARPS * STAGES * 2 * TILE;
    static constexpr int MERGE = 2 * (8 * NT * LD + 8 * NT * 4) * 4;            // two warps' rows, and their references
    static constexpr int SCALES = FEW_WARPS * STAGES * 2 * UNIT<HD> * 4;
    static constexpr int BYTES = RING + MERGE + SCALES + FEW_WARPS * STAGES * 8 + 16 + 64;                       // 64: Edge twice, and two answers
    static_assert(BLOCKS * (BYTES + 1024) <= 227 * 1024, "blocks of an SM");
};

// the physical row of a tile of 8 that stands for index g of the products: see the banks above
template <int HD> __device__ __forceinline__ int row_of(int g) {
    if (HD == 128) return g ^ ((g & 1) << 2);
    const int t = g >> 1, even = (t & 1) | ((t >> 1) << 2);
    return g & 1 ? even ^ 3 : even;
}
template <int HD> __device__ __forceinline__ int byte_of(int row, int chunk) {
    return HD == 128 ? row * 128 + ((chunk ^ (row & 7)) << 4) : row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
constexpr uint32_t BYTES_TO_F16 = 0x64806480u, MINUS_1152 = 0xe480e480u;
// bytes 0 and 2 (1 and 3) of x as two fp16 numbers, times s (with off = -1152 s)
// (one operation of three operands; written as (x & a) ^ b it was two)
__device__ __forceinline__ uint32_t biased(uint32_t x) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(d) : "r"(x), "r"(0x00ff00ffu), "r"(BYTES_TO_F16));
    return d;
}
__device__ __forceinline__ uint32_t even_bytes(uint32_t x, uint32_t s, uint32_t off) { return hfma2(biased(x), s, off); }
__device__ __forceinline__ uint32_t odd_bytes(uint32_t x, uint32_t s, uint32_t off) { return hfma2(biased(x >> 8), s, off); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
    return d;
}
__device__ __forceinline__ void cp_async4(void* smem, const void* global) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem_u32(smem)), "l"(global));
}
// 2^(exponent - most + SCALE_UP) for the exponents of two scales, 0 for those without one, as fp16 numbers (0 below what it holds)
__device__ __forceinline__ float power_of(int exponent, int most) { return exponent ? __uint_as_float((uint32_t)max(exponent - most + SCALE_UP + 127, 0) << 23) : 0.f; }
// How far a maximum of `from` (-inf: nothing yet) lies below one of `to`, which is no smaller
__device__ __forceinline__ float moved_by(float from, float to) { return from == -INFINITY ? -INFINITY : from - to; }
// 2^(a - b) for references that may be -inf (of nothing)
__device__ __forceinline__ float ratio(float a, float b) { return a == -INFINITY ? 0.f : fast_exp2(a - b); }

// The pages of a sequence that its rows see: places first .. first + pages - 1 of its table. 0 pages where it brings nothing or more than `most_tokens`,
// and where it does not fit (check_span).
struct Span {
    int first, pages, first_token, n_new, first_pos;
};
__device__ __forceinline__ Span span_of(const Args& a, int seq, int most_tokens) {
    Span s;
    s.first_token = a.cu_seqlens[seq];
    const int end = a.cu_seqlens[seq + 1];
    s.n_new = end - s.first_token;
    s.first_pos = a.seq_lens[seq] - s.n_new;
    s.first = first_seen(a, s.first_pos) / LLMB_PAGE;
    s.pages = pages_seen(a, s.first_pos, s.n_new);
    if (s.n_new <= 0 || s.n_new > most_tokens || s.first_token < 0 || end > a.n_tokens || s.first_pos < 0 || s.pages > a.ring_pages) s.pages = 0;
    return s;
}
// What does not fit is reported: places that there are not, more tokens than max_new says.
__device__ __forceinline__ void check_span(const Args& a, const Span& s, int* status) {
    if (s.n_new <= 0) return;
    if (s.first_token < 0 || s.first_token + s.n_new > a.n_tokens || s.first_pos < 0 || pages_seen(a, s.first_pos, s.n_new) > a.ring_pages) report(status, OUT_OF_RANGE);
    else if (s.n_new > a.max_new) report(status, BEYOND_BOUNDS);
}
// A (sequence, key head) pair and where its pages stand among all. (There are fewer than 2^31: a sequence has no more than its ring.)
struct Pair {
    int seq, head, start;
    Span span;
};
// The pages of all pairs, by every lane of a warp.
__device__ __forceinline__ int all_pages(const Args& a, int most_tokens, int lane) {
    int sum = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) sum += __reduce_add_sync(0xffffffffu, s0 + lane < a.n_seqs ? span_of(a, s0 + lane, most_tokens).pages : 0);
    return sum * a.n_kv_heads;
}
// The pair that page `at` of all belongs to.
__device__ __forceinline__ Pair pair_at(const Args& a, int at, int most_tokens, int lane) {
    int before = 0;
    Pair p;
    for (int s0 = 0;; s0 += 32) {
        const int mine = s0 + lane < a.n_seqs ? span_of(a, s0 + lane, most_tokens).pages : 0;
        int up = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            int left = __shfl_up_sync(0xffffffffu, up, d);
            if (lane >= d) up += left;
        }
        const unsigned beyond = __ballot_sync(0xffffffffu, at < before + up * a.n_kv_heads);
        if (beyond) {
            const int k = __ffs(beyond) - 1;
            p.seq = s0 + k;
            p.span = span_of(a, p.seq, most_tokens);
            p.start = before + (__shfl_sync(0xffffffffu, up, k) - p.span.pages) * a.n_kv_heads;
            p.head = (at - p.start) / p.span.pages;
            p.start += p.head * p.span.pages;
            return p;
        }
        before += __shfl_sync(0xffffffffu, up, 31) * a.n_kv_heads;
    }
}
// the pair behind it (there is one)
__device__ __forceinline__ void next_pair(const Args& a, Pair& p, int most_tokens) {
    p.start += p.span.pages;
    if (++p.head < a.n_kv_heads) return;
    p.head = 0;
    do p.span = span_of(a, ++p.seq, most_tokens); while (p.span.pages == 0 && p.seq + 1 < a.n_seqs);
}
// A block's range of `all` things that are dealt out to so many blocks, `least` at least.
__device__ __forceinline__ int range_of(int all, int blocks, int least) { return max((all + blocks - 1) / blocks, least); }
// The block that begins with something says which blocks have parts of it: x the first one, y how many.
__device__ __forceinline__ int2 blocks_of(int start, int count, int per) {
    const int first = start / per;
    return make_int2(first, (start + count - 1) / per - first + 1);
}

// A pair that the block has a part of, as the joining needs it.
struct Edge {
    int pair, start, pages, first_token, n_rows, out_column;
};
// A warp joins the parts of row r of a pair that blocks of.x .. of.x + of.y - 1 have, in their order whoever joins. (Read from L2: other blocks wrote them.)
template <int HD>
__device__ __forceinline__ void join_here(const float* acc, const float2* stats, int2 of, int r, __nv_bfloat16* to, int lane) {
    constexpr int W = HD / 32, AHEAD = 16;                     // a lane's columns, parts under way
    auto part_of = [&](int k) { return ((size_t)(of.x + k) * 2 + (k == 0 ? 1 : 0)) * FEW_ROWS + r; };
    float x[AHEAD][W], value[W], sum = 0.f, m = -INFINITY;
    auto fetch = [&](int k0) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
#pragma unroll
            for (int c = 0; c < W; ++c) x[j][c] = 0.f;
            if (k0 + j >= of.y) continue;
            const float* from = acc + part_of(k0 + j) * HD + lane * W;
            if constexpr (W == 4) *reinterpret_cast<float4*>(x[j]) = __ldcg(reinterpret_cast<const float4*>(from));
            else *reinterpret_cast<float2*>(x[j]) = __ldcg(reinterpret_cast<const float2*>(from));
        }
    };
#pragma unroll
    for (int c = 0; c < W; ++c) value[c] = 0.f;
    fetch(0);
    for (int k = lane; k < of.y; k += 32) m = fmaxf(m, __ldcg(stats + part_of(k)).x);
    m = warp_max(m);
    const float against = m == -INFINITY ? 0.f : m;
    for (int k0 = 0; k0 < of.y; k0 += 32) {
        const float2 st = k0 + lane < of.y ? __ldcg(stats + part_of(k0 + lane)) : make_float2(-INFINITY, 0.f);
        const float weight = st.y != 0.f ? exp2f(st.x - against) : 0.f;
        sum += st.y * weight;
        for (int j0 = 0; j0 < 32 && k0 + j0 < of.y; j0 += AHEAD) {
            if (k0 + j0) fetch(k0 + j0);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const float of_part = __shfl_sync(0xffffffffu, weight, j0 + j);
#pragma unroll
                for (int c = 0; c < W; ++c) value[c] = fmaf(x[j][c], of_part, value[c]);
            }
        }
    }
    sum = warp_sum(sum);
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int c = 0; c < W; c += 2) *reinterpret_cast<uint32_t*>(to + lane * W + c) = pack_bf16(value[c] * inv, value[c + 1] * inv);
}

template <int HD, int NT>
__global__ void __launch_bounds__(FEW_THREADS, Few<HD, NT>::BLOCKS)
attention_int8_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args a, int* status) {
    using F = Few<HD, NT>;
    constexpr int U = UNIT<HD>, TILE = F::TILE, STAGES = F::STAGES, LD = F::LD, DIMS = HD / 8, CHUNKS = HD / 64;     // DIMS: a lane's columns of the result
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* base = smem_raw;                            // (its alignment is the swizzle's)
    const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = base + warp * STAGES * 2 * TILE;
    float* merge = reinterpret_cast<float*>(base + F::RING);                     // [2] a warp's rows [8 NT][LD], then (m, R, l, -) of each
    float* scales = reinterpret_cast<float*>(base + F::RING + F::MERGE) + warp * STAGES * 2 * U;            // of this warp: [stage][2][U]
    uint64_t* full = reinterpret_cast<uint64_t*>(base + F::RING + F::MERGE + F::SCALES) + warp * STAGES;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(base + F::RING + F::MERGE + F::SCALES + FEW_WARPS * STAGES * 8);

    // the block's first pair, where another block begins it, and its last, where another one ends it; whether this block joins them
    Edge* edges = reinterpret_cast<Edge*>(base + F::RING + F::MERGE + F::SCALES + FEW_WARPS * STAGES * 8 + 16);
    int* joins = reinterpret_cast<int*>(edges + 2);
    griddep_launch();
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(smem_u32(&full[i]), 1);
        if (warp == 0) {
            *abort_flag = 0;
            edges[0].n_rows = edges[1].n_rows = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // (lengths, tables and the order are not written by the kernels of a step: a block finds its place before the kernel in front is done)
    const int share = a.n_heads / a.n_kv_heads, most_tokens = a.few_tokens;
    Pair pair;
    int r0, r1, per = 0;                                       // the block's range of all pages
    if (a.deal_blocks == 0) {                                  // a pair a block
        const int at = blockIdx.x / a.n_kv_heads;
        pair.seq = a.seq_order ? a.seq_order[at] : at;
        pair.head = blockIdx.x % a.n_kv_heads;
        pair.start = r0 = 0;
        const bool there = (unsigned)pair.seq < (unsigned)a.n_seqs;
        pair.span = span_of(a, there ? pair.seq : 0, most_tokens);
        r1 = there ? pair.span.pages : 0;
        if (threadIdx.x == 0) there ? check_span(a, pair.span, status) : report(status, OUT_OF_RANGE);
    } else {
        const int all = all_pages(a, most_tokens, lane);
        per = range_of(all, a.deal_blocks, a.deal_least);
        if (blockIdx.x == 0)
            for (int s = threadIdx.x; s < a.n_seqs; s += FEW_THREADS) {
                check_span(a, span_of(a, s, most_tokens), status);
                if (a.seq_order && (unsigned)a.seq_order[s] >= (unsigned)a.n_seqs) report(status, OUT_OF_RANGE);
            }
        r0 = min((long long)blockIdx.x * per, (long long)all);
        r1 = min(r0 + per, all);
        if (r0 < r1) pair = pair_at(a, r0, most_tokens, lane);
    }
    if (r0 >= r1) return griddep_wait();
    constexpr int PER_PAGE = LLMB_PAGE / U, TILES = U / 16;
    const int units = (r1 - r0) * PER_PAGE;
    const int scales_per_page = LLMB_PAGE >> a.block_shift;

    // What is asked for: unit `asked` of the range, of pair `ahead` (up to page `ahead_end` of the range); its page's number is on its way.
    Pair ahead = pair;
    int asked = warp, page_ahead = 0, ahead_end = pair.start - r0 + pair.span.pages;
    auto look_up = [&]() {
        if (asked >= units) return;
        const int at = asked / PER_PAGE;
        while (at >= ahead_end) {
            next_pair(a, ahead, most_tokens);
            ahead_end += ahead.span.pages;
        }
        page_ahead = page_at(a, a.block_table + (size_t)ahead.seq * a.table_stride, ahead.span.first + ahead.span.pages - (ahead_end - at), status);
    };
    auto ask = [&](int stage) {
        if (asked < units) {
            const int head_row = page_ahead * a.n_kv_heads + ahead.head, row = asked % PER_PAGE * U;
            float* to_scales = scales + stage * 2 * U + lane;
#pragma unroll
            for (int k = 0; k < U; k += 32) {
                const int at = head_row * scales_per_page + ((row + lane + k) >> a.block_shift);
                cp_async4(to_scales + k, a.key_scales + at);
                cp_async4(to_scales + U + k, a.value_scales + at);
            }
            if (elect_one()) {
                const uint32_t bar = smem_u32(&full[stage]), to = smem_u32(ring + stage * 2 * TILE);
                mbar_expect_tx(bar, 2 * TILE);
                tma_load_2d(to, &map_k, bar, 0, head_row * LLMB_PAGE + row);
                tma_load_2d(to + TILE, &map_v, bar, 0, head_row * LLMB_PAGE + row);
            }
            __syncwarp();
            asked += FEW_WARPS;
            look_up();
        }
        cp_async_commit();
    };
    look_up();
    griddep_wait();
#pragma unroll
    for (int i = 0; i < STAGES; ++i) ask(i);

    const __nv_bfloat16* q_all = behind_wait(static_cast<const __nv_bfloat16*>(a.q));
    int done = warp, stage = 0;                                // the next unit, and where it arrives
    uint32_t phase = 0;
    bool ok = true;
    const int my_row = row_of<HD>(g);
    for (;;) {
        // ---- the pair's rows
        const Span& span = pair.span;
        const int n_rows = span.n_new * share;
        const int pair_begin = pair.start - r0, pair_end = pair_begin + span.pages, range_end = r1 - r0;       // in pages of the range
        if (per && !a.arrived && pair_begin >= 0 && threadIdx.x == 0) a.few_blocks_of[pair.seq * a.n_kv_heads + pair.head] = blocks_of(pair.start, span.pages, per);
        const int end = min(pair_end, range_end);
        const int limit = span.first_pos + span.n_new - 1, low = first_seen(a, span.first_pos);       // positions that a row sees at all,
        const int all_to = span.first_pos, all_from = first_seen(a, limit);                           // and that all rows see
        uint32_t qb[NT][HD / 16][2];
        float row_scale[NT][2];                                // of rows 2t and 2t + 1 of each tile
        int pos[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = n * 8 + g;
            const bool valid = r < n_rows;
            const __nv_bfloat16* q = q_all + (size_t)(span.first_token + (valid ? r : 0) / share) * a.q_stride +
                                     (size_t)(pair.head * share + (valid ? r : 0) % share) * HD + 16 * t;
            uint4 raw[CHUNKS][2];
            uint32_t most = 0;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    raw[c][i] = valid ? *reinterpret_cast<const uint4*>(q + 64 * c + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t x[4] = {raw[c][i].x, raw[c][i].y, raw[c][i].z, raw[c][i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) most = max(most, max(x[k] & 0x7fffu, (x[k] >> 16) & 0x7fffu));
                }
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int exponent = max((int)(most >> 7), 27) - 127;                         // (rows below 2^-100 are as good as zero)
            const float factor = __uint_as_float((uint32_t)(14 - exponent + 127) << 23);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint4& v = raw[c][w >> 1];
                    const uint32_t x01 = w & 1 ? v.z : v.x, x23 = w & 1 ? v.w : v.y;       // columns 4w .. 4w + 3: two values each
                    const float x0 = __uint_as_float(x01 << 16) * factor, x1 = __uint_as_float(x01 & 0xffff0000u) * factor;
                    const float x2 = __uint_as_float(x23 << 16) * factor, x3 = __uint_as_float(x23 & 0xffff0000u) * factor;
                    qb[n][c * 4 + w][0] = pack_f16(x0, x2);
                    qb[n][c * 4 + w][1] = pack_f16(x1, x3);
                }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int of = n * 8 + 2 * t + j, e = __shfl_sync(0xffffffffu, exponent, (2 * t + j) * 4);
                row_scale[n][j] = a.scale_log2 * __uint_as_float((uint32_t)(max(e - 14 + 127, 1)) << 23);
                // (rows that are none have queries of zero and see everything: nothing is masked for them)
                pos[n][j] = of < n_rows ? span.first_pos + of / share : limit;
            }
        }
        float acc[NT][DIMS / 2][4], m[NT][2], lag[NT][2], sum[NT][2];            // lag: the reference, from the maximum
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < DIMS / 2; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[n][i][k] = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                m[n][j] = lag[n][j] = -INFINITY;
                sum[n][j] = 0.f;
            }
        }
        // ---- its units
        for (; done < end * PER_PAGE; done += FEW_WARPS) {
            const int key0 = (span.first + done / PER_PAGE - pair_begin) * LLMB_PAGE + done % PER_PAGE * U;
            ok = ok && mbar_wait_warp(smem_u32(&full[stage]), phase, abort_flag, status, 21);
            cp_async_wait<STAGES - 1>();
            __syncwarp();
            if (ok && key0 <= limit && key0 + U > low) {
                const unsigned char* k_tile = ring + stage * 2 * TILE;
                const unsigned char* v_tile = k_tile + TILE;
                // the unit's scales, a lane a position: the largest of those that are seen, then all as fp16 powers from it. (Blocks of 16 positions and
                // more have one for all 16 of a tile, and it counts where any of these is seen.)
                const int alike = a.block_shift >= 4 ? 15 : 0;
                uint32_t* packed = reinterpret_cast<uint32_t*>(scales + stage * 2 * U);       // (each lane's over its key's: key's low, value's high)
                uint32_t ks[U / 32], vs[U / 32], bad[U / 32], any_bad = 0;
                int ke = 0, ve = 0;
#pragma unroll
                for (int k = 0; k < U / 32; ++k) {
                    const int nearest = key0 + ((lane + 32 * k) & ~alike);
                    const bool seen = nearest <= limit && nearest + alike >= low;
                    ks[k] = seen ? packed[lane + 32 * k] : 0u;
                    vs[k] = seen ? packed[U + lane + 32 * k] : 0u;
                    const bool none = max(ks[k] & 0x7fffffffu, vs[k] & 0x7fffffffu) >= NOT_FINITE;
                    bad[k] = __ballot_sync(0xffffffffu, none);
                    any_bad |= bad[k];
                    if ((ks[k] | vs[k]) & 0x807fffffu && !none) report(status, NOT_A_POWER);
                    ks[k] = none ? 0u : ks[k] >> 23 & 0xffu;
                    vs[k] = none ? 0u : vs[k] >> 23 & 0xffu;
                    ke = max(ke, (int)ks[k]);
                    ve = max(ve, (int)vs[k]);
                }
                ke = __reduce_max_sync(0xffffffffu, ke);
                ve = __reduce_max_sync(0xffffffffu, ve);
#pragma unroll
                for (int k = 0; k < U / 32; ++k) packed[lane + 32 * k] = pack_f16(power_of((int)ks[k], ke), power_of((int)vs[k], ve));
                __syncwarp();

                float s[TILES][NT][4];
#pragma unroll
                for (int tile = 0; tile < TILES; ++tile) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) s[tile][n][k] = 0.f;
                    const int row = tile * 16 + my_row;
                    uint32_t sa = packed[row], sb = sa;        // of this position and the one 8 behind it
                    if (a.block_shift < 4) sb = packed[row + 8];
                    sa = __byte_perm(sa, 0, 0x1010);
                    sb = __byte_perm(sb, 0, 0x1010);
                    const uint32_t oa = hmul2(sa, MINUS_1152), ob = hmul2(sb, MINUS_1152);
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) {
                        const uint4 xa = *reinterpret_cast<const uint4*>(k_tile + byte_of<HD>(row, 4 * c + t));
                        const uint4 xb = *reinterpret_cast<const uint4*>(k_tile + byte_of<HD>(row + 8, 4 * c + t));
                        const uint32_t wa[4] = {xa.x, xa.y, xa.z, xa.w}, wb[4] = {xb.x, xb.y, xb.z, xb.w};
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t a0 = even_bytes(wa[w], sa, oa), a2 = odd_bytes(wa[w], sa, oa);
                            const uint32_t a1 = even_bytes(wb[w], sb, ob), a3 = odd_bytes(wb[w], sb, ob);
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_f16(s[tile][n], a0, a1, a2, a3, qb[n][c * 4 + w][0], qb[n][c * 4 + w][1]);
                        }
                    }
                }
                if (key0 + U - 1 > all_to || key0 < all_from || any_bad) {        // some rows do not see all of the unit
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int most = pos[n][j] - key0, least = first_seen(a, pos[n][j]) - key0;
#pragma unroll
                            for (int i = 0; i < 2 * TILES; ++i) {
                                float& x = s[i >> 1][n][(i & 1) * 2 + j];
                                const int at = my_row + 8 * i;
                                if (bad[(8 * i) / 32] >> (at & 31) & 1) x = __uint_as_float(0x7fffffffu);
                                if (at > most || at < least) x = -INFINITY;
                            }
                        }
                }
                const float k_unit = __uint_as_float((uint32_t)max(ke - SCALE_UP, 1) << 23);                  // what a step of the keys stands for
                const float v_unit = (float)(ve - 127);
                float top[NT][2];
                bool moved = false;
                // scores in base-2 units: rounded before the maximum is taken off, so that the largest is off by nothing whatever its size
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float c = fmaxf(row_scale[n][j] * k_unit, 1.1754944e-38f);
#pragma unroll
                        for (int i = 0; i < 2 * TILES; ++i) {
                            float& score = s[i >> 1][n][(i & 1) * 2 + j];
                            score = __fmul_rn(score, c);       // (a packed product would be joined with the packed sum below)
                        }
                        float x = fmaxf(s[0][n][j], s[0][n][2 + j]);
#pragma unroll
                        for (int tile = 1; tile < TILES; ++tile) x = max3(x, s[tile][n][j], s[tile][n][2 + j]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        top[n][j] = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        moved |= top[n][j] > m[n][j] || top[n][j] - m[n][j] + v_unit > lag[n][j];
                    }
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float new_m = fmaxf(m[n][j], top[n][j]), by = moved_by(m[n][j], new_m), held = lag[n][j] + by;
                            const float new_lag = fmaxf(held, moved_by(top[n][j], new_m) + v_unit);
                            sum[n][j] *= fast_exp2(by);
                            const float shrink = ratio(held, new_lag);
#pragma unroll
                            for (int i = 0; i < DIMS / 2; ++i) {
                                acc[n][i][j] *= shrink;
                                acc[n][i][2 + j] *= shrink;
                            }
                            m[n][j] = new_m;
                            lag[n][j] = new_lag;
                        }
                }
                uint32_t pb[TILES][NT][2];                     // the weights, positions on the contracted side
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float weight[TILES][4], against[2], lift[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        // (a row that has seen nothing yet has a maximum of -inf, and all its weights are zero)
                        against[j] = m[n][j] == -INFINITY ? 0.f : -m[n][j];
                        lift[j] = fast_exp2(fminf(v_unit + (float)WEIGHT_UP - lag[n][j], 126.f));
                    }
                    const uint64_t against2 = pair_of(against[0], against[1]), lift2 = pair_of(lift[0], lift[1]);
                    uint64_t sum2 = pair_of(sum[n][0], sum[n][1]);
#pragma unroll
                    for (int i = 0; i < 2 * TILES; ++i) {
                        const float(&x)[4] = s[i >> 1][n];
                        float p0, p1;
                        unpair(add2(pair_of(x[(i & 1) * 2], x[(i & 1) * 2 + 1]), against2), p0, p1);
                        const uint64_t p = pair_of(fast_exp2(p0), fast_exp2(p1));
                        sum2 = add2(sum2, p);                  // of this lane's positions
                        unpair(mul2(p, lift2), weight[i >> 1][(i & 1) * 2], weight[i >> 1][(i & 1) * 2 + 1]);
                    }
                    unpair(sum2, sum[n][0], sum[n][1]);
#pragma unroll
                    for (int tile = 0; tile < TILES; ++tile)
#pragma unroll
                        for (int half = 0; half < 2; ++half) pb[tile][n][half] = transposed(pack_f16(weight[tile][2 * half], weight[tile][2 * half + 1]));
                }
#pragma unroll
                for (int tile = 0; tile < TILES; ++tile) {
                    // positions 2t, 2t + 1 of the products, and 8 behind them
                    const int row[2] = {tile * 16 + row_of<HD>(2 * t), tile * 16 + row_of<HD>(2 * t + 1)};
                    uint32_t s_low, s_high;
                    if (a.block_shift >= 4) {
                        s_low = s_high = __byte_perm(packed[row[0]], 0, 0x3232);
                    } else {
                        s_low = __byte_perm(packed[row[0]], packed[row[1]], 0x7632);
                        s_high = __byte_perm(packed[row[0] + 8], packed[row[1] + 8], 0x7632);
                    }
                    const uint32_t o_low = hmul2(s_low, MINUS_1152), o_high = hmul2(s_high, MINUS_1152);
                    uint32_t x[4][DIMS / 4];                   // positions 2t, 2t + 1, 2t + 8, 2t + 9: this lane's columns
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int from = row[i & 1] + (i >> 1) * 8;
                        if constexpr (HD == 128) {
                            const uint4 v = *reinterpret_cast<const uint4*>(v_tile + byte_of<HD>(from, g));
                            x[i][0] = v.x;
                            x[i][1] = v.y;
                            x[i][2] = v.z;
                            x[i][3] = v.w;
                        } else {
                            const uint2 v = *reinterpret_cast<const uint2*>(v_tile + byte_of<HD>(from, g >> 1) + (g & 1) * 8);
                            x[i][0] = v.x;
                            x[i][1] = v.y;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < DIMS / 4; ++w)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {                  // columns 4w + 2 half, + 1
                            const uint32_t y_low = __byte_perm(x[0][w], x[1][w], half ? 0x7632 : 0x5410);
                            const uint32_t y_high = __byte_perm(x[2][w], x[3][w], half ? 0x7632 : 0x5410);
                            const uint32_t a0 = even_bytes(y_low, s_low, o_low), a1 = odd_bytes(y_low, s_low, o_low);
                            const uint32_t a2 = even_bytes(y_high, s_high, o_high), a3 = odd_bytes(y_high, s_high, o_high);
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_f16(acc[n][2 * w + half], a0, a1, a2, a3, pb[tile][n][0], pb[tile][n][1]);
                        }
                }
            }
            __syncwarp();                                      // everyone has read the unit: its room is free
            ask(stage);
            if (++stage == STAGES) {
                stage = 0;
                phase ^= 1;
            }
        }
        // ---- the four warps' sums, in a fixed order: 2 to 0 and 3 to 1, then 1 to 0
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                sum[n][j] += __shfl_xor_sync(0xffffffffu, sum[n][j], 4);
                sum[n][j] += __shfl_xor_sync(0xffffffffu, sum[n][j], 8);
                sum[n][j] += __shfl_xor_sync(0xffffffffu, sum[n][j], 16);
            }
        constexpr int HALF = 8 * NT * LD + 8 * NT * 4;
#pragma unroll
        for (int round = 0; round < 2; ++round) {
            const int from = 2 >> round;                       // warps from .. 2 from - 1 hand over to those `from` below
            float* rows = merge + (warp & (from - 1)) * HALF;
            __syncthreads();
            if (warp >= from && warp < 2 * from) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int r = n * 8 + 2 * t + j;
#pragma unroll
                        for (int i = 0; i < DIMS / 2; ++i)
                            *reinterpret_cast<float2*>(rows + r * LD + g * DIMS + 2 * i) = make_float2(acc[n][i][j], acc[n][i][2 + j]);
                        if (g == 0) *reinterpret_cast<float4*>(rows + 8 * NT * LD + r * 4) = make_float4(m[n][j], lag[n][j], sum[n][j], 0.f);
                    }
            }
            __syncthreads();
            if (warp < from) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int r = n * 8 + 2 * t + j;
                        const float4 other = *reinterpret_cast<const float4*>(rows + 8 * NT * LD + r * 4);
                        const float new_m = fmaxf(m[n][j], other.x), by = moved_by(m[n][j], new_m), other_by = moved_by(other.x, new_m);
                        const float held = lag[n][j] + by, other_held = other.y + other_by, new_lag = fmaxf(held, other_held);
                        sum[n][j] = sum[n][j] * fast_exp2(by) + other.z * fast_exp2(other_by);
                        const float mine = ratio(held, new_lag), theirs = ratio(other_held, new_lag);
#pragma unroll
                        for (int i = 0; i < DIMS / 2; ++i) {
                            const float2 x = *reinterpret_cast<const float2*>(rows + r * LD + g * DIMS + 2 * i);
                            acc[n][i][j] = acc[n][i][j] * mine + x.x * theirs;
                            acc[n][i][2 + j] = acc[n][i][2 + j] * mine + x.y * theirs;
                        }
                        m[n][j] = new_m;
                        lag[n][j] = new_lag;
                    }
            }
        }
        if (warp == 0) {
            const bool whole = pair_begin >= 0 && pair_end <= range_end;
            if (!whole && lane == 0)
                edges[pair_begin >= 0] = Edge{pair.seq * a.n_kv_heads + pair.head, pair.start, span.pages, span.first_token, n_rows, pair.head * share * HD};
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = n * 8 + 2 * t + j;
                    if (r >= n_rows) continue;
                    float factor = sum[n][j] != 0.f ? fast_exp2(lag[n][j] - (float)(WEIGHT_UP + SCALE_UP)) : 0.f;
                    if (whole) {
                        factor /= sum[n][j] != 0.f ? sum[n][j] : 1.f;
                        uint32_t out[DIMS / 2];
#pragma unroll
                        for (int i = 0; i < DIMS / 2; ++i) out[i] = pack_bf16(acc[n][i][j] * factor, acc[n][i][2 + j] * factor);
                        __nv_bfloat16* to = static_cast<__nv_bfloat16*>(a.out) + (size_t)(span.first_token + r / share) * a.out_stride +
                                            (size_t)(pair.head * share + r % share) * HD + g * DIMS;
#pragma unroll
                        for (int i = 0; i < DIMS / 2; i += 4) *reinterpret_cast<uint4*>(to + 2 * i) = make_uint4(out[i], out[i + 1], out[i + 2], out[i + 3]);
                    } else {
                        const size_t part = ((size_t)blockIdx.x * 2 + (pair.start >= r0 ? 1 : 0)) * FEW_ROWS + r;
                        float* to = a.acc + part * HD + g * DIMS;
#pragma unroll
                        for (int i = 0; i < DIMS / 2; i += 2)
                            *reinterpret_cast<float4*>(to + 2 * i) = make_float4(acc[n][i][j] * factor, acc[n][i][2 + j] * factor, acc[n][i + 1][j] * factor,
                                                                                 acc[n][i + 1][2 + j] * factor);
                        if (g == 0) *reinterpret_cast<float2*>(a.stats + part * 2) = make_float2(sum[n][j] != 0.f ? m[n][j] : -INFINITY, sum[n][j]);
                    }
                }
        }
        if (end >= range_end) break;
        next_pair(a, pair, most_tokens);
    }
    if (NT == 1 && a.arrived) {
        // the block whose part of a pair comes last joins all, and the count is zero again
        if (warp == 0) {
            __threadfence();
            __syncwarp();
            if (lane < 2) {
                const Edge& e = edges[lane];
                const unsigned last = blocks_of(e.start, e.pages, per).y - 1;
                joins[lane] = e.n_rows > 0 && atomicInc(reinterpret_cast<unsigned*>(a.arrived) + e.pair, last) == last;
            }
        }
        __syncthreads();
        for (int i = 0; i < 2; ++i) {
            if (!joins[i]) continue;
            __threadfence();
            const Edge e = edges[i];
            for (int r = warp; r < e.n_rows; r += FEW_WARPS)
                join_here<HD>(a.acc, reinterpret_cast<const float2*>(a.stats), blocks_of(e.start, e.pages, per), r,
                              static_cast<__nv_bfloat16*>(a.out) + (size_t)(e.first_token + r / share) * a.out_stride + e.out_column + r % share * HD, lane);
        }
    }
    __syncthreads();
    if (*abort_flag)                                           // a wait ran out: copies in flight get their time before the block leaves
        for (int i = 0; i < 100; ++i) __nanosleep(10000);
}

// The parts that several blocks have of a row: a row is one of `stride` of a (sequence, key head) pair, or of a pair's tile, `of` says which blocks. WARPS
// warps a row, each with every WARPS-th part; their sums are added in order.
constexpr int JOIN_WARPS = 8, JOIN_AHEAD = 4;
template <int HD, int WARPS>
__device__ __forceinline__ void join_row(const float* acc, const float2* stats, int2 of, int stride, int r, bool there, __nv_bfloat16* to) {
    constexpr int W = HD / 32;                                 // a lane's columns
    __shared__ float shared_value[JOIN_WARPS][HD];
    __shared__ float shared_sum[JOIN_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = warp % WARPS;
    auto part_of = [&](int k) { return ((size_t)(of.x + k) * 2 + (k == 0 ? 1 : 0)) * stride + r; };
    float value[W], sum = 0.f;
#pragma unroll
    for (int c = 0; c < W; ++c) value[c] = 0.f;
    if (there) {
        float m = -INFINITY;
        for (int k = lane; k < of.y; k += 32) m = fmaxf(m, stats[part_of(k)].x);
        for (int k0 = mine; k0 < of.y; k0 += WARPS * JOIN_AHEAD) {
            float x[JOIN_AHEAD][W];
            float2 st[JOIN_AHEAD];
#pragma unroll
            for (int j = 0; j < JOIN_AHEAD; ++j) {
                const int k = k0 + j * WARPS;
                st[j] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int c = 0; c < W; ++c) x[j][c] = 0.f;
                if (k < of.y) {
                    st[j] = stats[part_of(k)];
                    const float* from = acc + part_of(k) * HD + lane * W;
                    if constexpr (W == 4) *reinterpret_cast<float4*>(x[j]) = *reinterpret_cast<const float4*>(from);
                    else *reinterpret_cast<float2*>(x[j]) = *reinterpret_cast<const float2*>(from);
                }
            }
            if (k0 == mine) m = warp_max(m);                   // (the loads above are under way)
            const float against = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int j = 0; j < JOIN_AHEAD; ++j) {
                const float weight = st[j].y != 0.f ? exp2f(st[j].x - against) : 0.f;
                sum += st[j].y * weight;
#pragma unroll
                for (int c = 0; c < W; ++c) value[c] = fmaf(x[j][c], weight, value[c]);
            }
        }
    }
    if (WARPS > 1) {
#pragma unroll
        for (int c = 0; c < W; ++c) shared_value[warp][lane * W + c] = value[c];
        if (lane == 0) shared_sum[warp] = sum;
        __syncthreads();
        if (mine == 0)
#pragma unroll
            for (int k = 1; k < WARPS; ++k) {
                sum += shared_sum[warp + k];
#pragma unroll
                for (int c = 0; c < W; ++c) value[c] += shared_value[warp + k][lane * W + c];
            }
    }
    if (mine == 0 && there) {
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
        for (int c = 0; c < W; c += 2) *reinterpret_cast<uint32_t*>(to + lane * W + c) = pack_bf16(value[c] * inv, value[c + 1] * inv);
    }
}

template <int HD, int WARPS>
__global__ void __launch_bounds__(JOIN_WARPS * 32) attention_int8_few_join_kernel(const __grid_constant__ Args a, int rows) {
    griddep_launch();
    const int share = a.n_heads / a.n_kv_heads, most = a.few_tokens * share;      // rows of a pair
    const int row = blockIdx.x * (JOIN_WARPS / WARPS) + (threadIdx.x >> 5) / WARPS;
    const int pair = row / most, r = row - pair * most, seq = pair / a.n_kv_heads, head = pair - seq * a.n_kv_heads;
    Span span{};
    if (row < rows) span = span_of(a, seq, a.few_tokens);
    griddep_wait();
    bool there = span.pages > 0 && r < span.n_new * share;
    const int2 of = there ? behind_wait(a.few_blocks_of)[pair] : make_int2(0, 0);
    there = there && of.y > 1;                                 // (one block has finished it where it was worked on)
    join_row<HD, WARPS>(behind_wait(a.acc), reinterpret_cast<const float2*>(behind_wait(a.stats)), of, FEW_ROWS, r, there,
                        static_cast<__nv_bfloat16*>(a.out) + (size_t)(span.first_token + r / share) * a.out_stride + (size_t)(head * share + r % share) * HD);
}

// ------------------------------------------------------------------------------------------------ bfloat16, many rows
//
// 256 rows a block, one block an SM: two tiles of 128 rows with four softmax warps each share the keys and values of 128 positions (two pages). One warp
// has a step's bytes copied to shared memory and works out its scales, four widen them, as above, to the fp16 operands of the products (tcgen05), which
// another one issues. (Fetched through the widening warps' registers a step took 9,000 cycles: the fence between their stores and the products
// waits for their loads too.) Per tile one buffer of
// scores [128, 128] and O [128, D] fill tensor memory; the two tiles take turns: while the softmax of one works on its scores, the products of
// the other run (P V of these positions, then Q K^T of the next). Widening is a quarter of all instructions, and 256 rows share it.
//
// Four prompts of 120 to 510 tokens behind 16,384 positions take 380 us in short bursts (0.54 of the products' burst rate), 415 in long loops; a prompt of 2,048
// tokens 55. A step takes some 4,300 cycles; its products alone are 2,048, its exponentials as many on their unit, its instructions 2,560 of a
// scheduler's slots and its traffic through shared memory some 2,800.
//
// References as above, with two differences: keys' scales count from the largest of the 128 positions of a step, values' from the largest of each page (from
// 2^-90 of the largest so far at least, which keeps the sums of the weights exact where a page's values are zeros), and R moves only when it is exceeded by 2^8
// (weights below 2^-31 of the row's largest contribution may be lost).
//
// The steps of all (sequence, key head, tile), one after the other, are dealt out to the blocks in ranges of equal length, as pages are above; barriers
// and buffers run on from one tile to the next, so the next tile's keys are fetched and widened while a result is written.

constexpr int WIDE_THREADS = 768;           // warps 0 products, 1 pages and scales, 4-11 and 12-19 a tile's softmax (four for each page), 20-23 widening
constexpr int WIDE_ROWS = 256, TILE_ROWS = 128, STEP = 128, STEP_PAGES = STEP / LLMB_PAGE;
constexpr int TILE_PIECE = TILE_ROWS * 128, STEP_PIECE = STEP * 128;             // 64 columns of the head: 16 KB
constexpr int REGS_ISSUE = 72, REGS_SOFTMAX = 88, REGS_WIDEN = 56, REGS_LAUNCHED = 80;
static_assert(128 * (REGS_ISSUE + 4 * REGS_SOFTMAX + REGS_WIDEN) <= WIDE_THREADS * REGS_LAUNCHED, "the shares come from what the block is launched with");
constexpr int WIDE_UP = 7;                  // power of two that weights are lifted to; R may lag 2^8 behind
constexpr int VALUE_SPAN = 90;
constexpr float LARGEST_SCORE = 8388608.f;  // 2^23, in base-2 units: beyond, a reference (integers away from a score) is not exact and weights leave fp16; reported
constexpr int INFOS = 4;                    // steps whose scales are on their way to the softmax: the step behind the next one may be widened by then

struct StepInfo {
    float k_unit, v_unit[2];         // what a step of the keys stands for; exponent of the values' reference, of each page
    uint32_t any_bad;
    uint32_t bad[4];                 // positions whose scale is no number
};

// A tile of a (sequence, key head) and its pages.
struct Segment {
    int seq, head, tile;
    int row0, n_rows;
    int first_page, pages, steps;
    int low, limit;                  // positions that a row of the tile sees at all
    Span span;
    int start;                       // its first step among all
};
__device__ __forceinline__ int tiles_of(const Args& a, const Span& s) { return (s.n_new * (a.n_heads / a.n_kv_heads) + WIDE_ROWS - 1) / WIDE_ROWS; }
__device__ __forceinline__ void place_tile(const Args& a, Segment& g) {
    const int share = a.n_heads / a.n_kv_heads;
    g.row0 = g.tile * WIDE_ROWS;
    g.n_rows = min(WIDE_ROWS, g.span.n_new * share - g.row0);
    g.low = first_seen(a, g.span.first_pos + g.row0 / share);
    g.limit = g.span.first_pos + (g.row0 + g.n_rows - 1) / share;
    g.first_page = g.low / LLMB_PAGE;
    g.pages = g.limit / LLMB_PAGE + 1 - g.first_page;
    g.steps = (g.pages + STEP_PAGES - 1) / STEP_PAGES;
}
// The sequence as this kernel takes it: 0 pages where the kernel for few rows does, or nothing is brought.
__device__ __forceinline__ Span wide_span(const Args& a, int seq) {
    Span s = span_of(a, seq, a.max_new);
    if (s.n_new <= a.few_tokens) s.pages = 0;
    return s;
}
// Steps of a key head's tiles, one after the other, without a division for each (with them a prompt of 32 tiles took a block 40,000 cycles to find
// its place).
struct TileWalk {
    int tokens, rest;                // (tile * WIDE_ROWS) / share, and what is left
    int tile, tiles;
};
__device__ __forceinline__ TileWalk walk_of(const Args& a, const Span& s) { return TileWalk{0, 0, 0, s.pages > 0 ? tiles_of(a, s) : 0}; }
// the steps of the walk's tile; the walk goes on to the next
__device__ __forceinline__ int walk_steps(const Args& a, const Span& s, TileWalk& w, int share, int tokens, int rest) {
    const int low = first_seen(a, s.first_pos + w.tokens);
    w.tokens += tokens;
    w.rest += rest;
    if (w.rest >= share) {
        w.rest -= share;
        ++w.tokens;
    }
    const int last = ++w.tile == w.tiles ? s.n_new - 1 : w.rest ? w.tokens : w.tokens - 1;        // the tile's last token
    return ((s.first_pos + last) / LLMB_PAGE - low / LLMB_PAGE) / STEP_PAGES + 1;
}
// The steps of the first `most` tiles of one of the sequence's key heads.
__device__ __forceinline__ int steps_of(const Args& a, const Span& s, int most = 1 << 30) {
    const int share = a.n_heads / a.n_kv_heads, tokens = WIDE_ROWS / share, rest = WIDE_ROWS - tokens * share;
    int sum = 0;
    for (TileWalk w = walk_of(a, s); w.tile < min(w.tiles, most);) sum += walk_steps(a, s, w, share, tokens, rest);
    return sum;
}
__device__ __forceinline__ int all_steps(const Args& a, int lane) {
    int sum = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) sum += __reduce_add_sync(0xffffffffu, s0 + lane < a.n_seqs ? steps_of(a, wide_span(a, s0 + lane)) : 0);
    return sum * a.n_kv_heads;
}
__device__ __forceinline__ Segment segment_at(const Args& a, int at, int lane) {
    int before = 0;
    Segment g;
    for (int s0 = 0;; s0 += 32) {
        const int mine = s0 + lane < a.n_seqs ? steps_of(a, wide_span(a, s0 + lane)) : 0;
        int up = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            int left = __shfl_up_sync(0xffffffffu, up, d);
            if (lane >= d) up += left;
        }
        const unsigned beyond = __ballot_sync(0xffffffffu, at < before + up * a.n_kv_heads);
        if (beyond) {
            const int k = __ffs(beyond) - 1, steps = __shfl_sync(0xffffffffu, mine, k);
            g.seq = s0 + k;
            g.span = wide_span(a, g.seq);
            g.start = before + (__shfl_sync(0xffffffffu, up, k) - steps) * a.n_kv_heads;
            g.head = (at - g.start) / steps;
            g.start += g.head * steps;
            const int share = a.n_heads / a.n_kv_heads, tokens = WIDE_ROWS / share, rest = WIDE_ROWS - tokens * share;
            for (TileWalk w = walk_of(a, g.span);;) {
                g.tile = w.tile;
                const int here = walk_steps(a, g.span, w, share, tokens, rest);
                if (at < g.start + here) break;
                g.start += here;
            }
            place_tile(a, g);
            return g;
        }
        before += __shfl_sync(0xffffffffu, up, 31) * a.n_kv_heads;
    }
}
// the segment behind it (there is one)
__device__ __forceinline__ void next_segment(const Args& a, Segment& g) {
    g.start += g.steps;
    if (++g.tile >= tiles_of(a, g.span)) {
        g.tile = 0;
        if (++g.head == a.n_kv_heads) {
            g.head = 0;
            do g.span = wide_span(a, ++g.seq); while (g.span.pages == 0 && g.seq + 1 < a.n_seqs);
        }
    }
    place_tile(a, g);
}
// 8 bytes as 8 fp16 numbers times s (off = -1152 s), in their order
__device__ __forceinline__ uint4 widen8(uint2 v, uint32_t s, uint32_t off) {
    const uint32_t x = v.x ^ 0x80808080u, y = v.y ^ 0x80808080u;
    return make_uint4(hfma2(__byte_perm(x, 0x64646464u, 0x4140), s, off), hfma2(__byte_perm(x, 0x64646464u, 0x4342), s, off),
                      hfma2(__byte_perm(y, 0x64646464u, 0x4140), s, off), hfma2(__byte_perm(y, 0x64646464u, 0x4342), s, off));
}

template <int HD>
__global__ void __launch_bounds__(WIDE_THREADS, 1) attention_int8_wide_kernel(const __grid_constant__ Args a, int* status) {
    constexpr int PIECES = HD / 64, Q_BYTES = PIECES * TILE_PIECE, STEP_BYTES = PIECES * STEP_PIECE;
    constexpr uint32_t SCORES = 128, O_FIRST = 256, COLS = 512;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* q_tile = smem_raw;                         // [2]
    unsigned char* k_tile = q_tile + 2 * Q_BYTES;             // [2] steps
    unsigned char* v_tile = k_tile + 2 * STEP_BYTES;          // [2]
    unsigned char* raw_k = v_tile + 2 * STEP_BYTES;           // a step's bytes
    unsigned char* raw_v = raw_k + STEP * HD;
    StepInfo* infos = reinterpret_cast<StepInfo*>(raw_v + STEP * HD);            // [INFOS]
    unsigned short* step_scales = reinterpret_cast<unsigned short*>(infos + INFOS);      // [2][STEP] fp16 scales of the bytes' positions
    uint32_t* shared_rows = reinterpret_cast<uint32_t*>(step_scales + 2 * STEP);         // [tile][page][row] what the two warps of a row tell one another
    uint64_t* bars = reinterpret_cast<uint64_t*>(shared_rows + 4 * TILE_ROWS);
    uint64_t* q_full = bars;                  // [2] a tile's queries are in shared memory, its last result is out of tensor memory
    uint64_t* k_full = bars + 2;              // [2]
    uint64_t* k_empty = bars + 4;             // [2]
    uint64_t* v_full = bars + 6;              // [2]
    uint64_t* v_empty = bars + 8;             // [2]
    uint64_t* s_full = bars + 10;             // [2] a tile's scores are complete (and all its products before)
    uint64_t* p_full = bars + 12;             // [2][2] its weights of a page are written, and (with the first page's) O has been rescaled
    uint64_t* o_full = bars + 16;             // [2] the tile's last P V is complete
    uint64_t* raw_full = bars + 18;           // [2] a step's keys as bytes and their scales, its values and theirs
    uint64_t* raw_empty = bars + 20;          // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = warp_index(), lane = threadIdx.x & 31, share = a.n_heads / a.n_kv_heads;
    if (threadIdx.x == 0) {
#pragma unroll 1
        for (int i = 0; i < 22; ++i) {
            const bool by_all = i < 2 || i == 12 || i == 14;                      // a tile's eight warps; four below
            const bool by_group = i == 2 || i == 3 || i == 6 || i == 7 || i == 13 || i == 15 || i >= 20;
            mbar_init(smem_u32(&bars[i]), by_all ? 256 : by_group ? 128 : i >= 18 ? 2 : 1);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Tensor memory is taken when the kernel in front is done with it, and the next kernel may take some only when this one has it: two
    // that wait for one another's would stand still.
    griddep_wait();
    Segment segment;
    int r0, r1, per = 0;                                      // the block's range of all steps
    if (a.wide_blocks == 0) {                                 // a tile a block, those that see most first
        int x = blockIdx.x;
        segment.head = x % a.n_kv_heads;
        x /= a.n_kv_heads;
        const int back = x % a.tiles, at = x / a.tiles;
        segment.seq = a.seq_order ? a.seq_order[at] : at;
        if ((unsigned)segment.seq >= (unsigned)a.n_seqs) {
            if (threadIdx.x == 0) report(status, OUT_OF_RANGE);
            return;
        }
        segment.span = wide_span(a, segment.seq);
        if (threadIdx.x == 0 && back == 0) check_span(a, segment.span, status);
        const int tiles = segment.span.pages > 0 ? tiles_of(a, segment.span) : 0;
        if (back >= tiles) return;
        segment.tile = tiles - 1 - back;
        place_tile(a, segment);
        segment.start = r0 = 0;
        r1 = segment.steps;
    } else {
        const int all = all_steps(a, lane);
        per = range_of(all, a.wide_blocks, a.wide_least);
        if (blockIdx.x == 0)
            for (int s = threadIdx.x; s < a.n_seqs; s += WIDE_THREADS) {
                check_span(a, span_of(a, s, a.max_new), status);
                if (a.seq_order && (unsigned)a.seq_order[s] >= (unsigned)a.n_seqs) report(status, OUT_OF_RANGE);
            }
        r0 = min((long long)blockIdx.x * per, (long long)all);
        r1 = min(r0 + per, all);
        if (r0 >= r1) return;
        segment = segment_at(a, r0, lane);
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    griddep_launch();
    const uint32_t tmem_base = *tmem_slot;
    const int total = r1 - r0;                                // steps of the block, counted on over its segments
    // what the block has of a segment: its steps skip .. skip + count - 1
    auto share_of = [&](const Segment& g, int& skip, int& count) {
        skip = max(r0 - g.start, 0);
        count = min(g.start + g.steps, r1) - g.start - skip;
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_ISSUE));
        if (warp == 0) {
            // fp16 operands, 32-bit sums
            constexpr uint32_t idesc_qk = (1u << 4) | ((uint32_t)(STEP >> 3) << 17) | ((uint32_t)(TILE_ROWS >> 4) << 24);
            constexpr uint32_t idesc_pv = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(TILE_ROWS >> 4) << 24);
            const uint64_t q_desc = smem_desc(smem_u32(q_tile));
            const uint64_t k_desc0 = smem_desc(smem_u32(k_tile)), v_desc0 = smem_desc_mn(smem_u32(v_tile), STEP_PIECE);
            constexpr uint64_t BUFFER = (uint64_t)(STEP_BYTES >> 4), Q_TILE = (uint64_t)(Q_BYTES >> 4);
            uint32_t turns[2] = {0, 0}, segments[2] = {0, 0};  // of each tile so far
            auto issue_qk = [&](int tile, int n_tiles, int st) {
                const int b = st & 1;
                if (elect_one()) {
#pragma unroll
                    for (int j = 0; j < HD / 16; ++j) {
                        uint64_t q_off = (uint64_t)(((j >> 2) * TILE_PIECE + (j & 3) * 32) >> 4);
                        uint64_t k_off = (uint64_t)(((j >> 2) * STEP_PIECE + (j & 3) * 32) >> 4);
                        tcgen05_mma(tmem_base + tile * SCORES, q_desc + tile * Q_TILE + q_off, k_desc0 + b * BUFFER + k_off, idesc_qk, j > 0 ? 1u : 0u);
                    }
                    tcgen05_commit(smem_u32(&s_full[tile]));
                    if (tile == n_tiles - 1) tcgen05_commit(smem_u32(&k_empty[b]));
                }
                __syncwarp();
            };
            // the values of step st and the keys of the step behind it are in shared memory
            auto arrived = [&](int st, bool last) {
                return mbar_wait_warp(smem_u32(&v_full[st & 1]), (st >> 1) & 1, abort_flag, status, 36) &&
                       (last || mbar_wait_warp(smem_u32(&k_full[(st + 1) & 1]), ((st + 1) >> 1) & 1, abort_flag, status, 37));
            };
            // A tile's products of step st, then its scores of the next.
            auto turn = [&](int tile, int n_tiles, int st, bool first, bool last, bool last_but_one) -> bool {
                const int b = st & 1;
                const uint32_t o = tmem_base + O_FIRST + tile * HD, p = tmem_base + tile * SCORES;
#pragma unroll
                for (int half = 0; half < 2; ++half) {        // 64 positions each: the first are multiplied while the others' weights are formed
                    if (!mbar_wait_warp(smem_u32(&p_full[2 * tile + half]), turns[tile] & 1, abort_flag, status, 35)) return false;
                    tcgen05_fence_after();
                    // 16 positions a product: 8 columns of weights, 2048 bytes of value rows; a segment's first one overwrites O
                    if (elect_one()) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            tcgen05_mma_ts(o, p + half * LLMB_PAGE + j * 8, v_desc0 + b * BUFFER + (uint64_t)(((half * 4 + j) * 2048) >> 4), idesc_pv,
                                           first && half == 0 && j == 0 ? 0u : 1u);
                    }
                    __syncwarp();
                }
                ++turns[tile];
                if (elect_one()) {
                    if (last) tcgen05_commit(smem_u32(&o_full[tile]));
                    if (tile == n_tiles - 1) tcgen05_commit(smem_u32(&v_empty[b]));
                }
                __syncwarp();
                if (!last) {
                    issue_qk(tile, n_tiles, st + 1);
                    // the next keys and values are waited for where products are under way
                    if (tile == 0) return arrived(st + 1, last_but_one);
                }
                return true;
            };
            bool ok = true;
            for (int st = 0; st < total && ok;) {
                int skip, count;
                share_of(segment, skip, count);
                const int n_tiles = segment.n_rows > TILE_ROWS ? 2 : 1, end = st + count;
                ok = mbar_wait_warp(smem_u32(&k_full[st & 1]), (st >> 1) & 1, abort_flag, status, 34);
                for (int tile = 0; tile < n_tiles && ok; ++tile) {
                    ok = mbar_wait_warp(smem_u32(&q_full[tile]), segments[tile]++ & 1, abort_flag, status, 33);
                    if (!ok) break;
                    tcgen05_fence_after();
                    issue_qk(tile, n_tiles, st);
                }
                ok = ok && arrived(st, st + 1 == end);
                for (int i = st; i < end && ok; ++i) {
                    ok = turn(0, n_tiles, i, i == st, i + 1 == end, i + 2 == end);
                    if (n_tiles == 2) ok = ok && turn(1, n_tiles, i, i == st, i + 1 == end, false);
                }
                st = end;
                if (st < total) next_segment(a, segment);
            }
        } else if (warp == 1) {
            const int scales_per_page = LLMB_PAGE >> a.block_shift, alike = a.block_shift >= 4 ? 15 : 0;
            auto copy = [&](unsigned char* to, const signed char* from, uint64_t* bar, const int (&pages)[STEP_PAGES]) {
                if (elect_one()) {
                    mbar_expect_tx(smem_u32(bar), (pages[1] >= 0 ? 2 : 1) * LLMB_PAGE * HD);
#pragma unroll
                    for (int i = 0; i < STEP_PAGES; ++i)
                        if (pages[i] >= 0)
                            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                             smem_u32(to + i * LLMB_PAGE * HD)), "l"(from + (size_t)pages[i] * LLMB_PAGE * HD), "r"(LLMB_PAGE * HD), "r"(smem_u32(bar)) : "memory");
                }
                __syncwarp();
            };
            bool ok = true;
            for (int st = 0; st < total && ok;) {
                int skip, count;
                share_of(segment, skip, count);
                const int* table = a.block_table + (size_t)segment.seq * a.table_stride;
                int value_top = 0;                             // the largest exponent of the segment's values so far
                const int end = st + count;
                int next[STEP_PAGES];                          // the next step's page numbers are on their way
                auto look_up = [&](int i) {
#pragma unroll
                    for (int k = 0; k < STEP_PAGES; ++k) {
                        const int place = i * STEP_PAGES + k;
                        next[k] = place < segment.pages ? page_at(a, table, segment.first_page + place, status) * a.n_kv_heads + segment.head : -1;
                    }
                };
                look_up(skip);
                if (per && segment.start >= r0 && lane == 0)
                    a.wide_blocks_of[(segment.seq * a.n_kv_heads + segment.head) * a.tiles + segment.tile] = blocks_of(segment.start, segment.steps, per);
                for (int i = skip; st < end && ok; ++st, ++i) {
                    const int pages[STEP_PAGES] = {next[0], next[1]};
                    uint32_t ks[4], vs[4];                     // the scales of positions lane + 32 j of the step
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int page = pages[j >> 1], block = ((j & 1) * 32 + lane) >> a.block_shift;
                        ks[j] = page >= 0 ? __float_as_uint(a.key_scales[(size_t)page * scales_per_page + block]) : 0u;
                        vs[j] = page >= 0 ? __float_as_uint(a.value_scales[(size_t)page * scales_per_page + block]) : 0u;
                    }
                    if (st + 1 < end) look_up(i + 1);
                    ok = st == 0 || mbar_wait_warp(smem_u32(&raw_empty[0]), (st - 1) & 1, abort_flag, status, 43);
                    if (!ok) break;
                    copy(raw_k, a.keys, &raw_full[0], pages);
                    // scales from the largest of those that are seen
                    const int key0 = (segment.first_page + i * STEP_PAGES) * LLMB_PAGE;
                    StepInfo& info = infos[st % INFOS];
                    uint32_t bad[4];
                    int ke = 0, ve[STEP_PAGES] = {0, 0};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int nearest = key0 + ((lane + 32 * j) & ~alike);
                        const bool seen = nearest <= segment.limit && nearest + alike >= segment.low;
                        const uint32_t k = seen ? ks[j] : 0u, v = seen ? vs[j] : 0u;
                        const bool none = (k & 0x7fffffffu) >= NOT_FINITE || (v & 0x7fffffffu) >= NOT_FINITE;
                        if (!none && ((k | v) & 0x807fffffu)) report(status, NOT_A_POWER);
                        bad[j] = __ballot_sync(0xffffffffu, none);
                        ks[j] = none ? 0u : k >> 23 & 0xffu;
                        vs[j] = none ? 0u : v >> 23 & 0xffu;
                        ke = max(ke, (int)ks[j]);
                        ve[j >> 1] = max(ve[j >> 1], (int)vs[j]);
                    }
                    ke = __reduce_max_sync(0xffffffffu, ke);
#pragma unroll
                    for (int k = 0; k < STEP_PAGES; ++k) {
                        ve[k] = __reduce_max_sync(0xffffffffu, ve[k]);
                        value_top = max(value_top, ve[k]);
                        ve[k] = max(ve[k], value_top - VALUE_SPAN);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t both = pack_f16(power_of((int)ks[j], ke), power_of((int)vs[j], ve[j >> 1]));
                        step_scales[lane + 32 * j] = (unsigned short)both;
                        vs[j] = both >> 16;
                    }
                    if (lane == 0) {
                        info.k_unit = __uint_as_float((uint32_t)max(ke - SCALE_UP, 1) << 23);
                        info.v_unit[0] = (float)(ve[0] - 127);
                        info.v_unit[1] = (float)(ve[1] - 127);
                        info.any_bad = bad[0] | bad[1] | bad[2] | bad[3];
#pragma unroll
                        for (int j = 0; j < 4; ++j) info.bad[j] = bad[j];
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&raw_full[0]));
                    ok = st == 0 || mbar_wait_warp(smem_u32(&raw_empty[1]), (st - 1) & 1, abort_flag, status, 44);
                    if (!ok) break;
                    copy(raw_v, a.values, &raw_full[1], pages);
#pragma unroll
                    for (int j = 0; j < 4; ++j) step_scales[STEP + lane + 32 * j] = (unsigned short)vs[j];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&raw_full[1]));
                }
                if (st < total && ok) next_segment(a, segment);
            }
        }
    } else if (warp >= 20) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_WIDEN));
        // A pass is 16 bytes a thread. Of eight lanes four have half a row and four half of the next one: in the same columns where a row is 64 bytes,
        // the other half where it is 128, so that both what they read and the two chunks that each writes lie in different banks.
        constexpr int PASSES = HD / 16;
        const int t = threadIdx.x & 127, quad = t & 3, other = (t >> 2) & 1;
        bool ok = true;
        for (int i = 0; i < 2 * total && ok; ++i) {            // keys and values in turn
            const int st = i >> 1, which = i & 1, b = st & 1;
            uint64_t* full = bars + 2 + 4 * which + b;         // (k_full, v_full and their like)
            uint64_t* empty = bars + 4 + 4 * which + b;
            const unsigned short* scale = step_scales + which * STEP;
            const unsigned char* raw = which ? raw_v : raw_k;
            unsigned char* to = (which ? v_tile : k_tile) + b * STEP_BYTES;
            ok = mbar_wait_warp(smem_u32(&raw_full[which]), st & 1, abort_flag, status, 41) &&
                 (st < 2 || mbar_wait_warp(smem_u32(empty), ((st >> 1) - 1) & 1, abort_flag, status, 31));
            if (!ok) break;
            // rows to the operands' place, times their scales
#pragma unroll 1
            for (int i0 = 0; i0 < PASSES; i0 += 4) {
                uint4 x[4];
                uint32_t s[4];
                auto row_of_pass = [&](int j) { return HD == 128 ? (i0 + j) / 2 * 32 + t / 4 : (i0 + j) * 32 + t / 4; };
                auto piece_of_pass = [&](int j) { return HD == 128 ? (j & 1) ^ other : 0; };
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = row_of_pass(j);
                    x[j] = *reinterpret_cast<const uint4*>(raw + row * HD + piece_of_pass(j) * 64 + quad * 16);
                    s[j] = scale[row] * 0x10001u;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = row_of_pass(j);
                    const uint32_t off = hmul2(s[j], MINUS_1152);
                    unsigned char* at = to + piece_of_pass(j) * STEP_PIECE + row * 128;
                    *reinterpret_cast<uint4*>(at + (((2 * quad) ^ (row & 7)) << 4)) = widen8(make_uint2(x[j].x, x[j].y), s[j], off);
                    *reinterpret_cast<uint4*>(at + (((2 * quad + 1) ^ (row & 7)) << 4)) = widen8(make_uint2(x[j].z, x[j].w), s[j], off);
                }
            }
            mbar_arrive(smem_u32(&raw_empty[which]));          // the bytes' room is free
            fence_async_shared();
            mbar_arrive(smem_u32(full));
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
        // Two warps a row, one for each page of a step: they agree on the maximum, and each has its half of O's columns. (With one warp a row, 128 scores
        // one after the other, a step took 4,300 cycles; the loops stay short all the same.)
        const int tile = ((warp >> 2) - 1) >> 1, part = ((warp >> 2) - 1) & 1, quarter = warp & 3, r = quarter * 32 + lane;       // r: row of the tile = lane of tensor memory
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const uint32_t s_addr = lane_addr + tile * SCORES, o_addr = lane_addr + O_FIRST + tile * HD + part * (HD / 2);
        constexpr int PART_CHUNKS = HD / 16;                   // 16-byte chunks of this warp's half of a row of queries, or of a result on its way
        unsigned char* region = q_tile + tile * Q_BYTES + (HD == 128 ? part * TILE_PIECE : 0);
        auto place = [&](int row, int chunk) { return reinterpret_cast<uint4*>(region + row * 128 + (((chunk + (HD == 128 ? 0 : part * PART_CHUNKS)) ^ (row & 7)) << 4)); };
        uint32_t* mine = shared_rows + (tile * 2 + part) * TILE_ROWS + r;
        const uint32_t* theirs = shared_rows + (tile * 2 + 1 - part) * TILE_ROWS + r;
        auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + tile * 4 + quarter) : "memory"); };         // the two warps of these rows
        uint32_t turns = 0, segments = 0;
        bool ok = true;
        for (int st = 0; st < total;) {
            int skip, count;
            share_of(segment, skip, count);
            const int n_tiles = segment.n_rows > TILE_ROWS ? 2 : 1, end = st + count;
            const int tile_rows = segment.n_rows - tile * TILE_ROWS;        // of this tile, above 128 where it is full
            if (tile < n_tiles) {
                const bool valid = r < tile_rows, idle = quarter * 32 >= tile_rows;      // idle: a warp without rows (its lanes' weights reach nobody's result)
                const int at = segment.row0 + tile * TILE_ROWS + (valid ? r : 0);
                const int token = segment.span.first_token + at / share, head = segment.head * share + at % share;
                // (lanes without a row have queries of zero and see everything: nothing is masked for them)
                const int my_pos = valid ? segment.span.first_pos + at / share : 0x3fffffff, my_first = valid ? first_seen(a, my_pos) : 0;
                // The queries come row by row, the whole warp's at once; then each lane brings its row to fp16, the largest at 2^14, in place. (What is run
                // once a tile is written in short loops: its instructions are not at hand, and unrolled it took twice the time.)
                float row_scale;
                {
                    constexpr int ROWS = 32 / PART_CHUNKS;                       // rows to an instruction
                    const int chunk = lane % PART_CHUNKS;
                    const __nv_bfloat16* q = behind_wait(static_cast<const __nv_bfloat16*>(a.q)) + (size_t)(segment.head * share) * HD + part * (HD / 2) + chunk * 8;
                    int from = segment.row0 + tile * TILE_ROWS + quarter * 32 + lane / PART_CHUNKS, token0 = from / share, head0 = from - token0 * share;
                    token0 += segment.span.first_token;
#pragma unroll 2
                    for (int i = lane / PART_CHUNKS; i < 32; i += ROWS) {
                        const int row = quarter * 32 + i;
                        if (row < tile_rows) cp_async16(place(row, chunk), q + (size_t)token0 * a.q_stride + (size_t)head0 * HD);
                        else *place(row, chunk) = make_uint4(0u, 0u, 0u, 0u);
                        for (head0 += ROWS; head0 >= share; head0 -= share) ++token0;
                    }
                    cp_async_commit();
                    cp_async_wait<0>();
                    __syncwarp();
                    uint32_t most = 0;
#pragma unroll 2
                    for (int i = 0; i < PART_CHUNKS; ++i) {
                        const uint4 x = *place(r, i);
                        most = __vmaxu2(most, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
                    }
                    *mine = max(most & 0xffffu, most >> 16);
                    meet();
                    const int exponent = max((int)(max(*mine, *theirs) >> 7), 27) - 127;
                    const float factor = __uint_as_float((uint32_t)(14 - exponent + 127) << 23);
                    row_scale = a.scale_log2 * __uint_as_float((uint32_t)max(exponent - 14 + 127, 1) << 23);
#pragma unroll 2
                    for (int i = 0; i < PART_CHUNKS; ++i) {
                        const uint4 x = *place(r, i);
                        auto both = [&](uint32_t w) { return pack_f16(__uint_as_float(w << 16) * factor, __uint_as_float(w & 0xffff0000u) * factor); };
                        *place(r, i) = make_uint4(both(x.x), both(x.y), both(x.z), both(x.w));
                    }
                }
                fence_async_shared();
                tcgen05_fence_before();                        // (the last result has been read)
                mbar_arrive(smem_u32(&q_full[tile]));
                float run_max = -INFINITY, ref = -INFINITY, run_sum = 0.f, lowest = -INFINITY;      // lowest: the first maximum, as maxima only grow
                for (int i = st; i < end; ++i) {
                    ok = ok && mbar_wait_warp(smem_u32(&s_full[tile]), turns++ & 1, abort_flag, status, 38);
                    tcgen05_fence_after();
                    if (!ok) {                                 // (a wait has run out: the other warp of the rows may not know yet, and is met all the same)
                        if (!idle) meet();
                        continue;
                    }
                    if (idle) {
                        mbar_arrive(smem_u32(&p_full[2 * tile]));
                        if (part) mbar_arrive(smem_u32(&p_full[2 * tile + 1]));
                        continue;
                    }
                    const StepInfo& info = infos[i % INFOS];
                    const float c = fmaxf(row_scale * info.k_unit, 1.1754944e-38f);
                    const int key0 = (segment.first_page + (skip + i - st) * STEP_PAGES + part) * LLMB_PAGE;
                    const int last = my_pos - key0, first = my_first - key0;       // the positions of the page that the row sees
                    const uint32_t page_addr = s_addr + part * LLMB_PAGE;
                    const bool masked = __any_sync(0xffffffffu, last < LLMB_PAGE - 1 || first > 0) || info.any_bad;
                    float top = -INFINITY;
#pragma unroll 1
                    for (int from = 0; from < LLMB_PAGE; from += 32) {
                        uint32_t x[32];
                        tmem_ld32(page_addr + from, x);
                        if (masked) {                          // what the row does not see: -inf, in tensor memory too
                            const uint32_t bad = info.bad[2 * part + (from >> 5)];
                            const int most = last - from, least = first - from;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                if (bad >> j & 1) x[j] = 0x7fffffffu;
                                if (j > most || j < least) x[j] = __float_as_uint(-INFINITY);
                            }
                            tmem_st32(page_addr + from, x);
                        }
                        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            t0 = max3(t0, __uint_as_float(x[j]), __uint_as_float(x[j + 1]));
                            t1 = max3(t1, __uint_as_float(x[j + 2]), __uint_as_float(x[j + 3]));
                        }
                        top = max3(top, t0, t1);
                    }
                    tmem_st_wait();
                    top = __fmul_rn(top, c);                   // (not joined with a sum behind it: both warps of a row decide by the rounded one)
                    *mine = __float_as_uint(top);
                    meet();
                    const float other = __uint_as_float(*theirs);
                    const float new_max = max3(run_max, top, other), candidate = fmaxf(top + info.v_unit[part], other + info.v_unit[1 - part]);
                    // (a row that has seen no position yet keeps -inf, and all its weights are zero)
                    const bool move = candidate - ref > 8.f;
                    const float new_ref = move ? candidate : ref;
                    const float alpha = move ? fast_exp2(ref - new_ref) : 1.f;
                    const bool none = new_ref == -INFINITY;
                    const float shift = (none ? 0.f : (float)WIDE_UP - new_ref) + info.v_unit[part];
                    if (i > st && __any_sync(0xffffffffu, move)) {
#pragma unroll 1
                        for (int col = 0; col < HD / 2; col += 16) {
                            uint32_t o[16];
                            tmem_ld16(o_addr + col, o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                            tmem_st16(o_addr + col, o);
                        }
                        tmem_st_wait();
                    }
                    if (part) {                                // this half of O is ready for the first page's products
                        tcgen05_fence_before();
                        mbar_arrive(smem_u32(&p_full[2 * tile]));
                    }
                    const uint64_t scale2 = pair_of(c, c), shift2 = pair_of(shift, shift);
                    uint64_t add = pair_of(0u, 0u);
#pragma unroll 1
                    for (int from = 0; from < LLMB_PAGE; from += 32) {
                        uint32_t x[32], weights[16];
                        tmem_ld32(page_addr + from, x);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            float p0, p1;
                            unpair(fma2(pair_of(x[j], x[j + 1]), scale2, shift2), p0, p1);
                            p0 = fast_exp2(p0);
                            p1 = fast_exp2(p1);
                            add = add2(add, pair_of(p0, p1));
                            weights[j >> 1] = pack_f16(p0, p1);
                        }
                        tmem_st16(page_addr + from / 2, weights);      // over this page's scores that have been read
                    }
                    tmem_st_wait();
                    tcgen05_fence_before();
                    mbar_arrive(smem_u32(&p_full[2 * tile + part]));
                    float lo, hi;                              // what the page's weights are lifted by is taken off their sum
                    unpair(add, lo, hi);
                    run_sum = run_sum * ratio(run_max, new_max) + (none ? lo + hi : (lo + hi) * fast_exp2(-shift - new_max));
                    lowest = run_max == -INFINITY ? new_max : lowest;
                    run_max = new_max;
                    ref = new_ref;
                }
                // the result, or the block's part of it: by way of the queries' room, a warp's rows at a time, so that rows are written as a whole
                ok = ok && mbar_wait_warp(smem_u32(&o_full[tile]), segments++ & 1, abort_flag, status, 40);
                if (!ok && !idle) {
                    meet();
                    meet();
                } else if (!idle) {
                    tcgen05_fence_after();
                    *mine = __float_as_uint(run_sum);
                    meet();
                    run_sum += __uint_as_float(*theirs);
                    meet();                                    // (both have read)
                    const bool whole = segment.start >= r0 && segment.start + segment.steps <= r1;
                    if (valid && ((run_max > LARGEST_SCORE && run_max != INFINITY) || (lowest < -LARGEST_SCORE && lowest != -INFINITY))) report(status, LARGE_SCORES);
                    float factor = run_sum != 0.f ? fast_exp2(ref - (float)(WIDE_UP + SCALE_UP) - run_max) : 0.f;
                    const size_t row = ((size_t)blockIdx.x * 2 + (segment.start >= r0 ? 1 : 0)) * WIDE_ROWS + tile * TILE_ROWS + r;
                    unsigned char* to = nullptr;               // this half of the row in memory
                    if (whole) {
                        factor /= run_sum != 0.f ? run_sum : 1.f;
                        if (valid) to = reinterpret_cast<unsigned char*>(static_cast<__nv_bfloat16*>(a.out) + (size_t)token * a.out_stride + (size_t)head * HD + part * (HD / 2));
                    } else if (valid) {
                        to = reinterpret_cast<unsigned char*>(a.wide_acc + row * HD + part * (HD / 2));
                        if (part == 0) *reinterpret_cast<float2*>(a.wide_stats + row * 2) = make_float2(run_sum != 0.f ? run_max : -INFINITY, run_sum);
                    }
                    const int columns = whole ? HD / 2 : HD / 4;                 // that go out at a time: HD bytes
#pragma unroll 1
                    for (int from = 0; from < HD / 2; from += columns) {
#pragma unroll 1
                        for (int col = 0; col < columns; col += 16) {
                            uint32_t x[16];
                            tmem_ld16(o_addr + from + col, x);
#pragma unroll
                            for (int d = 0; d < 16; ++d) x[d] = __float_as_uint(__uint_as_float(x[d]) * factor);
                            if (whole) {
#pragma unroll
                                for (int d = 0; d < 16; d += 8)
                                    *place(r, (col + d) / 8) =
                                        make_uint4(pack2(__uint_as_float(x[d]), __uint_as_float(x[d + 1])), pack2(__uint_as_float(x[d + 2]), __uint_as_float(x[d + 3])),
                                                   pack2(__uint_as_float(x[d + 4]), __uint_as_float(x[d + 5])), pack2(__uint_as_float(x[d + 6]), __uint_as_float(x[d + 7])));
                            } else {
#pragma unroll
                                for (int d = 0; d < 16; d += 4) *place(r, (col + d) / 4) = make_uint4(x[d], x[d + 1], x[d + 2], x[d + 3]);
                            }
                        }
                        __syncwarp();
                        constexpr int ROWS = 32 / PART_CHUNKS;
                        const int chunk = lane % PART_CHUNKS;
#pragma unroll 2
                        for (int i = 0; i < 32; i += ROWS) {
                            const int from_row = i + lane / PART_CHUNKS;
                            unsigned char* there = reinterpret_cast<unsigned char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), from_row));
                            if (there) *reinterpret_cast<uint4*>(there + from * 4 + chunk * 16) = *place(quarter * 32 + from_row, chunk);
                        }
                        __syncwarp();
                    }
                }
            }
            st = end;
            if (st < total) next_segment(a, segment);
        }
    }

    tcgen05_fence_before();
    __syncthreads();
    if (*abort_flag) {                                         // a wait ran out: copies and products in flight get their time before the block leaves
        for (int i = 0; i < 100; ++i) __nanosleep(10000);
        __syncthreads();
    }
    if (warp == 0) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(COLS) : "memory");
    }
}

template <int HD, int WARPS>
__global__ void __launch_bounds__(JOIN_WARPS * 32) attention_int8_wide_join_kernel(const __grid_constant__ Args a) {
    griddep_launch();
    constexpr int ROWS = JOIN_WARPS / WARPS, BLOCKS = WIDE_ROWS / ROWS;          // of a block; of a tile
    const int share = a.n_heads / a.n_kv_heads, tile = blockIdx.x / BLOCKS, r = blockIdx.x % BLOCKS * ROWS + (threadIdx.x >> 5) / WARPS;
    Segment g;
    g.tile = tile % a.tiles;
    const int pair = tile / a.tiles;
    g.seq = pair / a.n_kv_heads;
    g.head = pair % a.n_kv_heads;
    g.span = wide_span(a, g.seq);
    const int at = g.tile * WIDE_ROWS + r;                     // the row of the sequence
    bool there = g.span.pages > 0 && at < g.span.n_new * share;
    griddep_wait();
    const int2 of = there ? behind_wait(a.wide_blocks_of)[tile] : make_int2(0, 0);
    there = there && of.y > 1;
    if (WARPS == 1 && !there) return;
    join_row<HD, WARPS>(behind_wait(a.wide_acc), reinterpret_cast<const float2*>(behind_wait(a.wide_stats)), of, WIDE_ROWS, r, there,
                        static_cast<__nv_bfloat16*>(a.out) + (size_t)(g.span.first_token + at / share) * a.out_stride + (size_t)(g.head * share + at % share) * HD);
}

// ------------------------------------------------------------------------------------------------ the parts joined
//
// WARPS warps a row: each reads all the maxima and sums, a lane two parts, and takes every WARPS-th part, several of them in flight; their
// sums are added in order. CHUNKS: 128 columns of the head each. Rows of tokens that no sequence has (a padded batch) have no parts, and are left as they are.
template <typename T, int WARPS, int CHUNKS>
__global__ void __launch_bounds__(256, CHUNKS == 1 ? 5 : 3) attention_int8_join_kernel(const __grid_constant__ Args a, int n_rows) {
    constexpr int ROWS = 8 / WARPS, AHEAD = 4;
    __shared__ float4 shared_value[8][CHUNKS * 32];
    griddep_launch();
    const int first_token = a.cu_seqlens[0], end_token = a.cu_seqlens[a.n_seqs];
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = warp % WARPS;
    const int row = blockIdx.x * ROWS + warp / WARPS, token = row / a.n_heads;
    const int D = a.head_dim, slots = a.slots, width = (D + 3) / 4;
    const bool valid = row < n_rows && token >= first_token && token < end_token, vectors = D % 4 == 0;
    float4 value[CHUNKS];
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) value[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (valid) {
        const float* acc = behind_wait(a.acc) + (size_t)row * slots * D;
        const float2* stats = reinterpret_cast<const float2*>(behind_wait(a.stats)) + (size_t)row * slots;
        static_assert(MAX_SPLITS <= 64, "two parts a lane");
        float2 part[2];
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            part[k] = lane + 32 * k < slots ? stats[lane + 32 * k] : make_float2(-INFINITY, 0.f);
            m = fmaxf(m, part[k].x);
        }
        m = warp_max(m);
        const float against = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            // (a part without keys has written no values; a sum that is no number stays none)
            part[k].x = part[k].y != 0.f ? exp2f(part[k].x - against) : 0.f;
            sum += part[k].x * part[k].y;
        }
        sum = warp_sum(sum);
        auto at = [&](int s, int c) {
            const int col = (c * 32 + lane) * 4;
            const float* from = acc + (size_t)s * D + col;
            if (vectors) return col < D ? *reinterpret_cast<const float4*>(from) : make_float4(0.f, 0.f, 0.f, 0.f);
            return make_float4(col < D ? from[0] : 0.f, col + 1 < D ? from[1] : 0.f, col + 2 < D ? from[2] : 0.f, col + 3 < D ? from[3] : 0.f);
        };
        for (int s0 = mine; s0 < slots; s0 += WARPS * AHEAD) {
            float weight[AHEAD];
            float4 x[AHEAD][CHUNKS];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int s = s0 + j * WARPS;
                weight[j] = __shfl_sync(0xffffffffu, s < 32 ? part[0].x : part[1].x, s & 31);
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
                    const float4 x = shared_value[warp + k][c * 32 + lane];
                    value[c].x += x.x;
                    value[c].y += x.y;
                    value[c].z += x.z;
                    value[c].w += x.w;
                }
    }
    if (!valid) return;
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    T* out = static_cast<T*>(a.out) + (size_t)token * a.out_stride + (size_t)(row % a.n_heads) * D;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int col = (c * 32 + lane) * 4;
        const float x[4] = {value[c].x * inv, value[c].y * inv, value[c].z * inv, value[c].w * inv};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (col + k < D) out[col + k] = from_float<T>(x[k]);
    }
}

// ------------------------------------------------------------------------------------------------ the launches

struct Sizes {
    int n_tokens, n_seqs, n_heads, n_kv_heads, head_dim, window, max_new, max_len;
    bool tc, alone;
};

struct Plan {
    bool few, wide;                  // which of the tensor-core kernels run (neither: the CUDA cores)
    int few_tokens;                  // sequences that bring at most so many tokens are the first one's
    long long few_blocks, wide_grid, blocks;
    int deal_blocks, deal_least, wide_blocks, wide_least;
    int rows;                        // of a block on the CUDA cores: 4 or 8 where a step has no more, 0: 32
    int tiles, slots;
    bool joins;                      // the kernel for few rows joins its parts itself
    long long part_rows, wide_rows;  // rows that are joined from parts
    int launches;
};

// The kernel for few rows deals pages out where a sequence may have more than WHOLE_PAGES, LEAST_PAGES a block at least. Below, a sequence and head are one
// block's, which saves the launch that joins, 4 us of the host's time: with 500 positions one sequence takes 8.3 us on the device, dealt out 7.7, 64
// take 20.1 and 20.8; with 1,000 positions one takes 13.5 and 8.0, 16 take 19.2 and 15.2.
constexpr int WHOLE_PAGES = 8, LEAST_PAGES = 4;
// The blocks join their parts themselves in calls outside of a step that is replayed, where a pair has up to 8 rows and no more than so many parts (a block joins
// one after another what a launch of its own spreads), and a block has no more than so many pages. A launch costs the host 2.5 us and, behind the kernel in a
// captured step, next to nothing; the end of a block, a fence, a count and the parts' way through L2 take 3. Calls one by one: eight sequences of 8,192
// positions (19 pages a block) take 35.8 us and with a launch 38.4, one 18.1 and 20.5, 64 (148 pages, all blocks end at once) 207 and 203. Captured: one 14.1 and
// 11.0, eight 38.2 and 37.7.
constexpr int JOIN_PARTS = 64, JOIN_PAGES = 48;
// The kernel for any shape cuts a sequence where it may have more pages than this.
constexpr int SIMT_WHOLE_PAGES = 4;
// The kernel for many rows deals steps out, LEAST_STEPS a block at least, unless no tile has more than WHOLE_STEPS.
constexpr int WHOLE_STEPS = 16, LEAST_STEPS = 4;

Plan plan_for(const Sizes& z) {
    Plan p = {};
    const int share = z.n_heads / z.n_kv_heads;
    const int seen = z.window > 0 && z.window + z.max_new < z.max_len ? z.window + z.max_new : z.max_len;
    const int pages = ceil_div(seen > 0 ? seen : 1, LLMB_PAGE);
    const long long pairs = (long long)z.n_seqs * z.n_kv_heads;
    p.slots = 1;
    p.launches = 1;
    if (z.tc) {
        p.few_tokens = FEW_ROWS / share < z.max_new ? FEW_ROWS / share : z.max_new;
        p.wide = (long long)z.max_new * share > FEW_ROWS;
        // sequences that bring few tokens beside others that bring many: there are some for certain only where the tokens are too few for all to bring more
        p.few = !p.wide || (p.few_tokens > 0 && z.n_tokens < (long long)z.n_seqs * (p.few_tokens + 1));
        if (!p.few) p.few_tokens = 0;
        p.launches = 0;
        if (p.few) {
            p.few_blocks = pairs;
            ++p.launches;
            if (pages > WHOLE_PAGES) {
                const long long held = SMS * ((long long)p.few_tokens * share <= 8 ? 3 : 2), most = ceil_div(pages, LEAST_PAGES) * pairs;
                p.deal_least = LEAST_PAGES;
                p.deal_blocks = (int)(most < held ? most : held);
                p.few_blocks = p.deal_blocks;
                p.part_rows = 2ll * p.deal_blocks * FEW_ROWS;
                p.joins = z.alone && (long long)p.few_tokens * share <= 8 && p.deal_blocks <= JOIN_PARTS * z.n_kv_heads && pages * pairs <= (long long)JOIN_PAGES * p.deal_blocks;
                if (!p.joins) ++p.launches;
            }
        }
        if (p.wide) {
            p.tiles = ceil_div((long long)z.max_new * share, WIDE_ROWS);
            p.wide_grid = pairs * p.tiles;
            ++p.launches;
            if (ceil_div(pages, STEP_PAGES) > WHOLE_STEPS) {
                p.wide_blocks = SMS;
                p.wide_least = LEAST_STEPS;
                p.wide_grid = SMS;
                p.wide_rows = 2ll * SMS * WIDE_ROWS;
                ++p.launches;
            }
        }
        return p;
    }
    p.rows = (long long)z.max_new * share <= 4 ? 4 : (long long)z.max_new * share <= 8 ? 8 : 0;
    if (p.rows) {
        // a page for each of a block's warps at least, as many slices as make two blocks an SM
        p.tiles = 1;
        p.blocks = pairs;
        const long long slots = 2ll * SMS / pairs, most = ceil_div(pages, ROWS_WARPS);
        p.slots = (int)(slots < 1 ? 1 : slots > most ? most : slots);
        if (p.slots > MAX_SPLITS) p.slots = MAX_SPLITS;
        p.part_rows = p.slots == 1 ? 0 : (long long)z.n_tokens * z.n_heads;
        if (p.slots > 1) ++p.launches;
        return p;
    }
    // Into how many slices the pages are cut: as many as make all blocks come to about the blocks that the SMs hold at once, two pages each at least; up
    // to SIMT_WHOLE_PAGES are one block's, since joining takes a launch.
    p.tiles = ceil_div((long long)z.max_new * share, SIMT_ROWS);
    p.blocks = pairs * p.tiles;
    const long long wave = (long long)SMS * (z.head_dim <= 128 ? 2 : 1);
    long long slots = wave / p.blocks;
    if (slots > pages / 2) slots = pages / 2;
    if (pages <= SIMT_WHOLE_PAGES) slots = 1;
    p.slots = slots < 1 ? 1 : slots > MAX_SPLITS ? MAX_SPLITS : (int)slots;
    p.part_rows = p.slots == 1 ? 0 : (long long)z.n_tokens * z.n_heads;
    if (p.slots > 1) ++p.launches;
    return p;
}

// of the parts' weighted values (their maxima and sums start on 16 bytes behind them), and of both
long long value_floats(long long parts, int head_dim) { return (parts * head_dim + 3) / 4 * 4; }
long long scratch_floats_of(long long parts, int head_dim) { return value_floats(parts, head_dim) + 2 * parts; }
// and of what says which blocks have them
long long places_of(const Plan& p, const Sizes& z) {
    const long long pairs = (long long)z.n_seqs * z.n_kv_heads;
    return (p.deal_blocks && !p.joins ? pairs : 0) + (p.wide_blocks ? pairs * p.tiles : 0);
}

// A kernel's shared memory is a setting of each device.
constexpr int MAX_DEVICES = 64;
int allow_shared(const void* kernel, size_t bytes, bool (&done)[MAX_DEVICES]) {
    int device = 0;
    LLMB_CUDA(cudaGetDevice(&device));
    if (device < MAX_DEVICES && done[device]) return LLMB_OK;
    LLMB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (device < MAX_DEVICES) done[device] = true;
    return LLMB_OK;
}

template <typename T, int DMAX>
int launch_simt(const Args& a, const Plan& p, int* status, cudaStream_t stream) {
    constexpr size_t smem = simt_floats<DMAX>() * sizeof(float);
    static bool done[MAX_DEVICES] = {};
    if (int code = allow_shared((const void*)attention_int8_simt_kernel<T, DMAX>, smem, done)) return code;
    llmb::launch(attention_int8_simt_kernel<T, DMAX>, dim3((unsigned)p.blocks, p.slots), SIMT_THREADS, smem, stream, true, a, status);
    return check_launch("attention_int8_simt");
}

template <typename T, int DMAX, int R>
int launch_rows(const Args& a, const Plan& p, int* status, cudaStream_t stream) {
    constexpr size_t smem = rows_floats<DMAX, R>() * sizeof(float);
    static bool done[MAX_DEVICES] = {};
    if (int code = allow_shared((const void*)attention_int8_rows_kernel<T, DMAX, R>, smem, done)) return code;
    llmb::launch(attention_int8_rows_kernel<T, DMAX, R>, dim3((unsigned)p.blocks, p.slots), ROWS_THREADS, smem, stream, true, a, status);
    return check_launch("attention_int8_rows");
}
template <typename T, int DMAX>
int launch_cores(const Args& a, const Plan& p, int* status, cudaStream_t stream) {
    return p.rows == 4 ? launch_rows<T, DMAX, 4>(a, p, status, stream) : p.rows == 8 ? launch_rows<T, DMAX, 8>(a, p, status, stream)
                                                                                    : launch_simt<T, DMAX>(a, p, status, stream);
}

// a warp for four parts, as many as fit
template <typename T, int CHUNKS>
void launch_join(const Args& a, int rows, cudaStream_t stream) {
    if (a.slots <= 4) llmb::launch(attention_int8_join_kernel<T, 1, CHUNKS>, dim3((rows + 7) / 8), 256, 0, stream, true, a, rows);
    else if (a.slots <= 8) llmb::launch(attention_int8_join_kernel<T, 2, CHUNKS>, dim3((rows + 3) / 4), 256, 0, stream, true, a, rows);
    else if (a.slots <= 16) llmb::launch(attention_int8_join_kernel<T, 4, CHUNKS>, dim3((rows + 1) / 2), 256, 0, stream, true, a, rows);
    else llmb::launch(attention_int8_join_kernel<T, 8, CHUNKS>, dim3(rows), 256, 0, stream, true, a, rows);
}

// 8-bit rows of a cache, boxes of a unit of them
int make_map_int8(CUtensorMap* map, const void* ptr, long long rows, int dim) {
    EncodeTiled encode = encode_fn();
    if (!encode) return fail(LLMB_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)dim};
    cuuint32_t box[2] = {(cuuint32_t)dim, (cuuint32_t)(dim == 64 ? UNIT<64> : UNIT<128>)}, elem[2] = {1, 1};
    CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LLMB_ERR_CUDA, "cuTensorMapEncodeTiled (8 bits) failed with %d", (int)r);
    return LLMB_OK;
}

template <int HD, int NT>
int launch_few(const Args& a, const Plan& p, int* status, cudaStream_t stream) {
    static bool done[MAX_DEVICES] = {};
    if (int code = allow_shared((const void*)attention_int8_few_kernel<HD, NT>, Few<HD, NT>::BYTES, done)) return code;
    CUtensorMap map_k, map_v;
    const long long rows = (long long)a.n_pages * a.n_kv_heads * LLMB_PAGE;
    int code = make_map_int8(&map_k, a.keys, rows, HD);
    if (!code) code = make_map_int8(&map_v, a.values, rows, HD);
    if (code) return code;
    llmb::launch(attention_int8_few_kernel<HD, NT>, dim3((unsigned)p.few_blocks), FEW_THREADS, Few<HD, NT>::BYTES, stream, true, map_k, map_v, a, status);
    if ((code = check_launch("attention_int8_few")) || p.deal_blocks == 0 || p.joins) return code;
    // as many warps a row as there is room for: a few rows have many parts each
    const int joined = a.n_seqs * a.n_kv_heads * a.few_tokens * (a.n_heads / a.n_kv_heads);
    if (joined <= 4 * SMS) llmb::launch(attention_int8_few_join_kernel<HD, 8>, dim3(joined), JOIN_WARPS * 32, 0, stream, true, a, joined);
    else if (joined <= 16 * SMS) llmb::launch(attention_int8_few_join_kernel<HD, 2>, dim3((joined + 3) / 4), JOIN_WARPS * 32, 0, stream, true, a, joined);
    else llmb::launch(attention_int8_few_join_kernel<HD, 1>, dim3((joined + 7) / 8), JOIN_WARPS * 32, 0, stream, true, a, joined);
    return check_launch("attention_int8_few_join");
}

template <int HD>
int launch_wide(const Args& a, const Plan& p, int* status, cudaStream_t stream) {
    // (more than half of an SM's shared memory for the smaller head size too: tensor memory has room for one block)
    constexpr size_t need = (HD / 64) * (2 * TILE_PIECE + 4 * STEP_PIECE) + 2 * STEP * HD + INFOS * sizeof(StepInfo) + 4 * STEP + 16 * TILE_ROWS + 23 * 8, bytes = need < 120 * 1024 ? 120 * 1024 : need;
    static_assert(bytes <= 227 * 1024, "one block an SM");
    static bool done[MAX_DEVICES] = {};
    static bool checked = false;
    if (!checked) {                              // (its softmax warps would wait for registers that are not there)
        cudaFuncAttributes built;
        LLMB_CUDA(cudaFuncGetAttributes(&built, attention_int8_wide_kernel<HD>));
        LLMB_REQUIRE(built.numRegs >= REGS_LAUNCHED, "attention_int8: built with %d registers a thread", built.numRegs);
        checked = true;
    }
    if (int code = allow_shared((const void*)attention_int8_wide_kernel<HD>, bytes, done)) return code;
    llmb::launch(attention_int8_wide_kernel<HD>, dim3((unsigned)p.wide_grid), WIDE_THREADS, bytes, stream, true, a, status);
    if (int code = check_launch("attention_int8_wide")) return code;
    if (p.wide_blocks == 0) return LLMB_OK;
    const unsigned tiles = (unsigned)a.n_seqs * a.n_kv_heads * a.tiles;
    if (tiles <= 32) llmb::launch(attention_int8_wide_join_kernel<HD, 4>, dim3(tiles * (WIDE_ROWS / 2)), JOIN_WARPS * 32, 0, stream, true, a);
    else llmb::launch(attention_int8_wide_join_kernel<HD, 1>, dim3(tiles * (WIDE_ROWS / JOIN_WARPS)), JOIN_WARPS * 32, 0, stream, true, a);
    return check_launch("attention_int8_wide_join");
}

template <int HD>
int launch_tc(const Args& a, const Plan& p, int* status, cudaStream_t stream) {
    int code = LLMB_OK;
    if (p.few) code = a.few_tokens * (a.n_heads / a.n_kv_heads) <= 8 ? launch_few<HD, 1>(a, p, status, stream) : launch_few<HD, 2>(a, p, status, stream);
    return code || !p.wide ? code : launch_wide<HD>(a, p, status, stream);
}

template <typename T>
int run(const Args& a, const Plan& p, const Sizes& z, int* status, cudaStream_t stream) {
    if (p.few || p.wide) return a.head_dim == 64 ? launch_tc<64>(a, p, status, stream) : launch_tc<128>(a, p, status, stream);
    int code = a.head_dim <= 64 ? launch_cores<T, 64>(a, p, status, stream) : a.head_dim <= 128 ? launch_cores<T, 128>(a, p, status, stream)
                                                                                                : launch_cores<T, 256>(a, p, status, stream);
    if (code || a.slots == 1) return code;
    if (a.head_dim <= 128) launch_join<T, 1>(a, (int)p.part_rows, stream);
    else launch_join<T, 2>(a, (int)p.part_rows, stream);
    return check_launch("attention_int8_join");
}

}  // namespace

LLMB_EXPORT int llmb_attention_int8_status() {
    int* s = status_word();
    if (!s) return -1;
    int v = *s;
    *s = 0;
    return v;
}

// The sizes of a call, one integer each.
struct llmb_int8_sizes {
    int q_stride, out_stride, table_stride, ring_pages, n_pages;    // elements between rows, pages of the caches
    int dtype, n_tokens, n_seqs, n_heads, n_kv_heads, head_dim, block, window;
    int max_new, max_len;                                           // upper bounds (ops.attention_int8)
    int tc;                                                         // whether the tensor-core kernels take the call (refused where they cannot), 0: the CUDA cores
    int alone;                                                      // the call is no part of a step that is replayed: a launch costs the host its time
};

namespace {
Sizes sizes_of(const llmb_int8_sizes& z) {
    return Sizes{z.n_tokens, z.n_seqs, z.n_heads, z.n_kv_heads, z.head_dim, z.window, z.max_new, z.max_len, z.tc != 0, z.alone != 0};
}
bool sane(const llmb_int8_sizes& z) {
    return z.n_tokens > 0 && z.n_seqs > 0 && z.n_kv_heads > 0 && z.n_heads > 0 && z.n_heads % z.n_kv_heads == 0 && z.max_new > 0 && z.max_len > 0 &&
           z.head_dim > 0;
}
}  // namespace

// Floats of scratch that a call of these sizes needs, the number of its launches in counts[0] and of its counters in counts[1].
LLMB_EXPORT long long llmb_attention_int8_scratch_floats(const llmb_int8_sizes* z, int* counts) {
    counts[0] = 1;
    counts[1] = 0;
    if (!sane(*z)) return 0;
    const Plan p = plan_for(sizes_of(*z));
    counts[0] = p.launches;
    counts[1] = p.joins ? z->n_seqs * z->n_kv_heads : 0;
    return scratch_floats_of(p.part_rows * p.slots + p.wide_rows, z->head_dim) + 2 * places_of(p, sizes_of(*z));
}

LLMB_EXPORT int llmb_attention_int8(const void* q, const void* keys, const float* key_scales, const void* values, const float* value_scales,
                                    const int* block_table, const int* seq_lens, const int* cu_seqlens, const int* seq_order, void* out, float* scratch,
                                    long long scratch_floats, int* arrived, int n_arrived, float scale, const llmb_int8_sizes* sizes, cudaStream_t stream) {
    const llmb_int8_sizes& z = *sizes;
    if (z.n_tokens == 0 || z.n_seqs == 0) return LLMB_OK;
    LLMB_REQUIRE(z.dtype == LLMB_DTYPE_F32 || z.dtype == LLMB_DTYPE_BF16, "attention_int8: float32 and bfloat16 are built");
    LLMB_REQUIRE(sane(z), "attention_int8: bad sizes (%d tokens, %d sequences, %d heads over %d of %d, at most %d new and %d positions)", z.n_tokens, z.n_seqs,
                 z.n_heads, z.n_kv_heads, z.head_dim, z.max_new, z.max_len);
    LLMB_REQUIRE(z.head_dim <= LLMB_MAX_HEAD_DIM && z.head_dim % 2 == 0, "attention_int8: head_dim %d (served: even, up to %d)", z.head_dim, LLMB_MAX_HEAD_DIM);
    int shift = 0;
    while (shift < 6 && (1 << shift) < z.block) ++shift;
    LLMB_REQUIRE(z.block == 1 << shift, "attention_int8: blocks of %d positions", z.block);
    LLMB_REQUIRE(z.window >= 0 && z.ring_pages > 0 && z.n_pages > 0, "attention_int8: window %d, ring of %d pages of %d", z.window, z.ring_pages, z.n_pages);
    LLMB_REQUIRE((long long)z.n_tokens * z.n_heads < (1ll << 31), "attention_int8: %d tokens of %d heads", z.n_tokens, z.n_heads);
    auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    LLMB_REQUIRE(aligned(keys) && aligned(values), "attention_int8: pages must start on 16 bytes");
    LLMB_REQUIRE(!z.tc || (z.dtype == LLMB_DTYPE_BF16 && (z.head_dim == 64 || z.head_dim == 128) && scale > 0.f && z.q_stride % 8 == 0 &&
                           z.out_stride % 8 == 0 && aligned(q) && aligned(out) && (long long)z.n_pages * z.n_kv_heads * LLMB_PAGE < (1ll << 31)),
                 "attention_int8: the tensor-core kernels do not take these operands");
    const Sizes s = sizes_of(z);
    const Plan p = plan_for(s);
    const long long pairs = (long long)z.n_seqs * z.n_kv_heads;
    LLMB_REQUIRE(p.blocks < (1ll << 31) && p.few_blocks < (1ll << 31) && p.wide_grid < (1ll << 31) && pairs * p.tiles * (WIDE_ROWS / 2) < (1ll << 31) &&
                 pairs * FEW_ROWS < (1ll << 31), "attention_int8: too many blocks");
    LLMB_REQUIRE(!z.tc || pairs * z.ring_pages * (p.wide ? p.tiles : 1) < (1ll << 31), "attention_int8: too many pages to deal out");
    const long long parts = p.part_rows * p.slots, all_parts = parts + p.wide_rows;
    LLMB_REQUIRE(all_parts == 0 || (scratch != nullptr && aligned(scratch) && scratch_floats >= scratch_floats_of(all_parts, z.head_dim) + 2 * places_of(p, s)),
                 "attention_int8: scratch too small");
    LLMB_REQUIRE(!p.joins || (arrived && n_arrived >= pairs), "attention_int8: %d counters for %lld sequences' heads", n_arrived, pairs);
    static int* status = nullptr;                // (one address for all devices)
    if (!status && status_word()) LLMB_CUDA(cudaHostGetDevicePointer((void**)&status, status_word(), 0));
    float* stats = scratch + value_floats(all_parts, z.head_dim);
    int2* places = reinterpret_cast<int2*>(stats + 2 * all_parts);
    const Args a{q, (const signed char*)keys, key_scales, (const signed char*)values, value_scales, block_table, seq_lens, cu_seqlens, seq_order, out, scratch,
                 stats, z.q_stride, z.out_stride, z.table_stride, z.ring_pages, z.n_pages, z.n_tokens, z.n_seqs, z.n_heads, z.n_kv_heads, z.head_dim,
                 shift, z.window, scale * LOG2E, z.max_new, p.tiles, p.slots, p.few_tokens, p.deal_blocks, p.deal_least, p.wide_blocks, p.wide_least,
                 scratch + parts * z.head_dim, stats + 2 * parts, places, places + (p.deal_blocks && !p.joins ? pairs : 0),
                 p.joins ? arrived : nullptr};
    return z.dtype == LLMB_DTYPE_F32 ? run<float>(a, p, s, status, stream) : run<__nv_bfloat16>(a, p, s, status, stream);
}

LLMB_PACKED(llmb_attention_int8)
