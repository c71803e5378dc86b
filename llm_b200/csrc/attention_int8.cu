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
};

// What a kernel reports (no wait has these codes): a step that brings more tokens than max_new says; a place outside of what the call was given, which is
// not read: a page, a token or a sequence that there is not.
constexpr int BEYOND_BOUNDS = 50, OUT_OF_RANGE = 51;
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
    if (w.first_token < 0 || end_token > a.n_tokens || (n_new > 0 && w.first_pos < 0)) {
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
    const int page = pages[logical % a.ring_pages];
    if ((unsigned)page < (unsigned)a.n_pages) return page;
    report(status, OUT_OF_RANGE);
    return 0;
}
// the first key that a position sees
__device__ __forceinline__ int first_seen(const Args& a, int position) { return a.window > 0 ? max(position - a.window + 1, 0) : 0; }

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
                bad[j] = is_number(k_scales[b]) && is_number(v_scales[b]) ? 0.f : __uint_as_float(0x7fffffffu);
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

// ------------------------------------------------------------------------------------------------ the parts joined
//
// WARPS warps a row: each reads all the maxima and sums, a lane two parts, and takes every WARPS-th part, several of them in flight; their
// sums are added in order. CHUNKS: 128 columns of the head each.
template <typename T, int WARPS, int CHUNKS>
__global__ void __launch_bounds__(256, CHUNKS == 1 ? 5 : 3) attention_int8_join_kernel(const __grid_constant__ Args a, int n_rows) {
    constexpr int ROWS = 8 / WARPS, AHEAD = 4;
    __shared__ float4 shared_value[8][CHUNKS * 32];
    griddep_launch();
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = warp % WARPS;
    const int row = blockIdx.x * ROWS + warp / WARPS;
    const int D = a.head_dim, slots = a.slots, width = (D + 3) / 4;
    const bool valid = row < n_rows, vectors = D % 4 == 0;
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
    T* out = static_cast<T*>(a.out) + (size_t)(row / a.n_heads) * a.out_stride + (size_t)(row % a.n_heads) * D;
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

struct Plan {
    int tiles, slots;
    long long blocks;                // of a slot
    long long part_rows;             // rows that are joined from parts
};

struct Sizes {
    int n_tokens, n_seqs, n_heads, n_kv_heads, head_dim, window, max_new, max_len;
    bool tc;
};

// Into how many slices the pages are cut: as many as make all blocks come to about the blocks that the SMs hold at once, two pages each at least.
Plan plan_for(const Sizes& z) {
    Plan p;
    const int share = z.n_heads / z.n_kv_heads;
    const int seen = z.window > 0 && z.window + z.max_new < z.max_len ? z.window + z.max_new : z.max_len;
    const int pages = ceil_div(seen > 0 ? seen : 1, LLMB_PAGE);
    p.tiles = ceil_div((long long)z.max_new * share, SIMT_ROWS);
    p.blocks = (long long)z.n_seqs * p.tiles * z.n_kv_heads;
    const long long wave = (long long)SMS * (z.head_dim <= 128 ? 2 : 1);
    long long slots = wave / p.blocks;
    if (slots > pages / 2) slots = pages / 2;
    p.slots = slots < 1 ? 1 : slots > MAX_SPLITS ? MAX_SPLITS : (int)slots;
    p.part_rows = p.slots == 1 ? 0 : (long long)z.n_tokens * z.n_heads;
    return p;
}

// of the parts' weighted values (their maxima and sums start on 16 bytes behind them), and of both
long long value_floats(long long parts, int head_dim) { return (parts * head_dim + 3) / 4 * 4; }
long long scratch_floats_of(long long parts, int head_dim) { return value_floats(parts, head_dim) + 2 * parts; }

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

// a warp for four parts, as many as fit
template <typename T, int CHUNKS>
void launch_join(const Args& a, int rows, cudaStream_t stream) {
    if (a.slots <= 4) llmb::launch(attention_int8_join_kernel<T, 1, CHUNKS>, dim3((rows + 7) / 8), 256, 0, stream, true, a, rows);
    else if (a.slots <= 8) llmb::launch(attention_int8_join_kernel<T, 2, CHUNKS>, dim3((rows + 3) / 4), 256, 0, stream, true, a, rows);
    else if (a.slots <= 16) llmb::launch(attention_int8_join_kernel<T, 4, CHUNKS>, dim3((rows + 1) / 2), 256, 0, stream, true, a, rows);
    else llmb::launch(attention_int8_join_kernel<T, 8, CHUNKS>, dim3(rows), 256, 0, stream, true, a, rows);
}

template <typename T>
int run(const Args& a, const Plan& p, const Sizes& z, int* status, cudaStream_t stream) {
    int code = a.head_dim <= 64 ? launch_simt<T, 64>(a, p, status, stream) : a.head_dim <= 128 ? launch_simt<T, 128>(a, p, status, stream)
                                                                                               : launch_simt<T, 256>(a, p, status, stream);
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
};

namespace {
Sizes sizes_of(const llmb_int8_sizes& z) {
    return Sizes{z.n_tokens, z.n_seqs, z.n_heads, z.n_kv_heads, z.head_dim, z.window, z.max_new, z.max_len, z.tc != 0};
}
bool sane(const llmb_int8_sizes& z) {
    return z.n_tokens > 0 && z.n_seqs > 0 && z.n_kv_heads > 0 && z.n_heads > 0 && z.n_heads % z.n_kv_heads == 0 && z.max_new > 0 && z.max_len > 0 &&
           z.head_dim > 0;
}
}  // namespace

// Floats of scratch that a call of these sizes needs, and the number of its launches in *kernels.
LLMB_EXPORT long long llmb_attention_int8_scratch_floats(const llmb_int8_sizes* z, int* kernels) {
    *kernels = 1;
    if (!sane(*z)) return 0;
    const Plan p = plan_for(sizes_of(*z));
    if (p.slots > 1) ++*kernels;
    return scratch_floats_of(p.part_rows * p.slots, z->head_dim);
}

LLMB_EXPORT int llmb_attention_int8(const void* q, const void* keys, const float* key_scales, const void* values, const float* value_scales,
                                    const int* block_table, const int* seq_lens, const int* cu_seqlens, const int* seq_order, void* out, float* scratch,
                                    long long scratch_floats, float scale, const llmb_int8_sizes* sizes, cudaStream_t stream) {
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
    const Sizes s = sizes_of(z);
    const Plan p = plan_for(s);
    LLMB_REQUIRE(p.blocks < (1ll << 31), "attention_int8: too many blocks");
    const long long parts = p.part_rows * p.slots;
    LLMB_REQUIRE(parts == 0 || (scratch != nullptr && aligned(scratch) && scratch_floats >= scratch_floats_of(parts, z.head_dim)),
                 "attention_int8: scratch too small");
    int* status = nullptr;
    if (status_word()) LLMB_CUDA(cudaHostGetDevicePointer((void**)&status, status_word(), 0));
    const Args a{q, (const signed char*)keys, key_scales, (const signed char*)values, value_scales, block_table, seq_lens, cu_seqlens, seq_order, out, scratch,
                 scratch + value_floats(parts, z.head_dim), z.q_stride, z.out_stride, z.table_stride, z.ring_pages, z.n_pages, z.n_tokens, z.n_seqs,
                 z.n_heads, z.n_kv_heads, z.head_dim, shift, z.window, scale * LOG2E, z.max_new, p.tiles, p.slots};
    return z.dtype == LLMB_DTYPE_F32 ? run<float>(a, p, s, status, stream) : run<__nv_bfloat16>(a, p, s, status, stream);
}

LLMB_PACKED(llmb_attention_int8)
