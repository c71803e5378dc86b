// Attention of a batch whose sequences share their first pages of the cache: several samples of one prompt, several questions
// behind one document. Sequences that stand together in the batch form groups; the members of a group have the same pages in the
// first `group_pages` places of their page tables. The keys and values of those pages are read once for all queries of the group.
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
// bounds (most tokens of a group, most pages) and a block beyond the real work leaves. A key beyond a row's position has no
// weight whatever is stored there, and values beyond a tile's last position are taken for zero, so that what an earlier sequence
// left in a page (infinities and NaN too) does not reach a result. A row that sees no key is zero.
#include "common.cuh"

using namespace llmb;

LLMB_DEFINE_LAST_ERROR(llmb_prefix_attention)

namespace {

constexpr float LOG2E = 1.4426950408889634f;

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
    float* acc;                      // [tokens * heads, slots, head_dim]
    float* stats;                    // [tokens * heads, slots, 2]: maximum in base-2 units, sum
    int q_stride, out_stride, table_stride, n_seqs, n_groups, n_heads, n_kv_heads, head_dim;
    float scale_log2;
    int prefix_tiles, prefix_splits, own_tiles, own_splits, slots;
    int vectors;                     // the caches' rows and the queries can be read 16 bytes at a time
};

// A block's share of the work: rows of a range of tokens against a slice of pages.
struct Item {
    int kv_head, tile, tiles, slot;
    int seq_first, seq_last;         // the sequences whose tokens are the rows
    int first_token, n_rows;
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
    int prefix_blocks = a.n_groups * a.prefix_tiles * a.prefix_splits;
    int share = a.n_heads / a.n_kv_heads;
    if (x < prefix_blocks) {
        w.tiles = a.prefix_tiles;
        w.tile = x % w.tiles;
        x /= w.tiles;
        int split = x % a.prefix_splits, group = x / a.prefix_splits;
        w.seq_first = a.group_first[group];
        w.seq_last = a.group_first[group + 1];
        int pages = a.group_pages[group], per = (pages + a.prefix_splits - 1) / a.prefix_splits;
        w.page_begin = min(split * per, pages);
        w.page_end = min(w.page_begin + per, pages);
        w.slot = split;
    } else {
        x -= prefix_blocks;
        w.tiles = a.own_tiles;
        w.tile = x % w.tiles;
        x /= w.tiles;
        int split = x % a.own_splits, seq = x / a.own_splits;
        w.seq_first = seq;
        w.seq_last = seq + 1;
        int first = a.group_pages[group_of(a, seq)], last = (a.seq_lens[seq] + LLMB_PAGE - 1) / LLMB_PAGE;
        int pages = max(last - first, 0), per = (pages + a.own_splits - 1) / a.own_splits;
        w.page_begin = first + min(split * per, pages);
        w.page_end = first + min(split * per + per, pages);
        w.slot = a.prefix_splits + split;
    }
    if (w.seq_first >= w.seq_last) return false;
    w.first_token = a.cu_seqlens[w.seq_first];
    w.n_rows = (a.cu_seqlens[w.seq_last] - w.first_token) * share;
    return true;
}

// the position of a token of the item's sequences
__device__ __forceinline__ int position_of(const Args& a, const Item& w, int token) {
    int low = w.seq_first, high = w.seq_last - 1;             // the last sequence whose tokens do not start behind this one
    while (low < high) {
        int mid = (low + high + 1) >> 1;
        if (a.cu_seqlens[mid] <= token) low = mid;
        else high = mid - 1;
    }
    return a.seq_lens[low] - a.cu_seqlens[low + 1] + token;
}

// ------------------------------------------------------------------------------------------------ any type, any head size
//
// 32-bit arithmetic on the CUDA cores: the path of 32-bit caches, and of the head sizes that the tensor-core kernel is not built for.
// A block holds 32 rows and walks its pages one by one: 64 keys and values in shared memory (as 32-bit values), thread
// (ty, tx) of a half-warp ty owns rows 4 ty .. 4 ty + 3. It forms their scores with keys tx, tx + 16, tx + 32, tx + 48 (4 x 4 products a
// pair of 16-byte loads), shares maxima and sums with the 15 other threads of its rows, and adds the weighted values of columns
// 4 tx + 64 c. Rows of a key or value are 4 words longer than the head, so that the 16 rows that a half-warp reads lie in
// different banks.

constexpr int SIMT_ROWS = 32, SIMT_THREADS = 128;

template <int DMAX>
constexpr int simt_floats() { return (SIMT_ROWS + 2 * LLMB_PAGE) * (DMAX + 4) + SIMT_ROWS * (LLMB_PAGE + 4) + SIMT_ROWS; }

template <typename T, int DMAX>
__global__ void __launch_bounds__(SIMT_THREADS) prefix_attention_simt_kernel(const __grid_constant__ Args a) {
    constexpr int LD = DMAX + 4, LP = LLMB_PAGE + 4, COLS = DMAX / 64;
    extern __shared__ __align__(16) float smem[];
    float* qs = smem;                              // [32][LD], scaled
    float* ks = qs + SIMT_ROWS * LD;               // [64][LD]
    float* vs = ks + LLMB_PAGE * LD;               // [64][LD]
    float* ps = vs + LLMB_PAGE * LD;               // [32][LP]
    int* row_pos = reinterpret_cast<int*>(ps + SIMT_ROWS * LP);

    griddep_launch();
    griddep_wait();
    Item w;
    if (!item_of(a, blockIdx.x, w)) return;
    const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
    const int D = a.head_dim, share = a.n_heads / a.n_kv_heads;
    const T* q = static_cast<const T*>(a.q);
    const T* k_cache = static_cast<const T*>(a.k_cache);
    const T* v_cache = static_cast<const T*>(a.v_cache);
    const int* pages = a.block_table + (size_t)w.seq_first * a.table_stride;

    for (int tile = w.tile; tile * SIMT_ROWS < w.n_rows; tile += w.tiles) {
        int row0 = tile * SIMT_ROWS, rows = min(SIMT_ROWS, w.n_rows - row0);
        __syncthreads();                           // the tile before is done with shared memory
        for (int i = tid; i < SIMT_ROWS * DMAX; i += SIMT_THREADS) {
            int r = i / DMAX, d = i - r * DMAX;
            float value = 0.f;
            if (r < rows && d < D) {
                int token = w.first_token + (row0 + r) / share, head = w.kv_head * share + (row0 + r) % share;
                value = to_float(q[(size_t)token * a.q_stride + (size_t)head * D + d]) * a.scale_log2;
            }
            qs[r * LD + d] = value;
        }
        if (tid < SIMT_ROWS) row_pos[tid] = tid < rows ? position_of(a, w, w.first_token + (row0 + tid) / share) : -1;
        __syncthreads();
        int last = -1;                             // the last position that a row of the tile sees
        for (int r = 0; r < rows; ++r) last = max(last, row_pos[r]);
        int end = min(w.page_end, last < 0 ? 0 : last / LLMB_PAGE + 1);

        float m[4], l[4], o[4][COLS * 4];
        int pos[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
            pos[i] = row_pos[ty * 4 + i];
#pragma unroll
            for (int c = 0; c < COLS * 4; ++c) o[i][c] = 0.f;
        }
        for (int logical = w.page_begin; logical < end; ++logical) {
            size_t base = ((size_t)pages[logical] * a.n_kv_heads + w.kv_head) * LLMB_PAGE * D;
            int key0 = logical * LLMB_PAGE, stored = min(LLMB_PAGE, last + 1 - key0);
            __syncthreads();                       // everyone is done with the page before
            constexpr int V = 16 / sizeof(T);
            if (a.vectors) {
                int per_row = D / V;
                for (int i = tid; i < LLMB_PAGE * per_row; i += SIMT_THREADS) {
                    int row = i / per_row, col = (i - row * per_row) * V;
                    __align__(16) T kk[V], vv[V];
                    *reinterpret_cast<uint4*>(kk) = *reinterpret_cast<const uint4*>(k_cache + base + (size_t)row * D + col);
                    *reinterpret_cast<uint4*>(vv) = *reinterpret_cast<const uint4*>(v_cache + base + (size_t)row * D + col);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        ks[row * LD + col + j] = to_float(kk[j]);
                        vs[row * LD + col + j] = row < stored ? to_float(vv[j]) : 0.f;
                    }
                }
            } else {
                int width = (D + 3) & ~3;          // (the scores read four columns at a time)
                for (int i = tid; i < LLMB_PAGE * width; i += SIMT_THREADS) {
                    int row = i / width, col = i - row * width;
                    bool in = col < D;
                    ks[row * LD + col] = in ? to_float(k_cache[base + (size_t)row * D + col]) : 0.f;
                    vs[row * LD + col] = in && row < stored ? to_float(v_cache[base + (size_t)row * D + col]) : 0.f;
                }
            }
            __syncthreads();
            if (ty * 4 >= rows) continue;          // (the same answer in a half-warp, whose threads alone share the rows)
            unsigned mates = 0xffffu << (tid & 16);

            float s[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
            for (int d = 0; d < D; d += 4) {
                float4 qv[4], kv[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(qs + (ty * 4 + i) * LD + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * LD + d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        s[i][j] = fmaf(qv[i].x, kv[j].x, fmaf(qv[i].y, kv[j].y, fmaf(qv[i].z, kv[j].z, fmaf(qv[i].w, kv[j].w, s[i][j]))));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (key0 + tx + 16 * j > pos[i]) s[i][j] = -INFINITY;
                    top = fmaxf(top, s[i][j]);
                }
#pragma unroll
                for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(mates, top, x));
                float new_m = fmaxf(m[i], top), against = new_m == -INFINITY ? 0.f : new_m;
                float alpha = exp2f(m[i] - against);
                m[i] = new_m;
                float add = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float p = exp2f(s[i][j] - against);
                    add += p;
                    ps[(ty * 4 + i) * LP + tx + 16 * j] = p;
                }
                l[i] = l[i] * alpha + add;         // of this thread's keys
#pragma unroll
                for (int c = 0; c < COLS * 4; ++c) o[i][c] *= alpha;
            }
            __syncwarp(mates);
            for (int j = 0; j < LLMB_PAGE; j += 4) {
                float4 pv[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pv[i] = *reinterpret_cast<const float4*>(ps + (ty * 4 + i) * LP + j);
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    if (c * 64 + tx * 4 >= D) break;
#pragma unroll
                    for (int jj = 0; jj < 4; ++jj) {
                        float4 v = *reinterpret_cast<const float4*>(vs + (j + jj) * LD + c * 64 + tx * 4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float p = jj == 0 ? pv[i].x : jj == 1 ? pv[i].y : jj == 2 ? pv[i].z : pv[i].w;
                            o[i][c * 4] = fmaf(p, v.x, o[i][c * 4]);
                            o[i][c * 4 + 1] = fmaf(p, v.y, o[i][c * 4 + 1]);
                            o[i][c * 4 + 2] = fmaf(p, v.z, o[i][c * 4 + 2]);
                            o[i][c * 4 + 3] = fmaf(p, v.w, o[i][c * 4 + 3]);
                        }
                    }
                }
            }
            __syncwarp(mates);                     // the weights are read before the next page's are written
        }
        if (ty * 4 < rows) {
            unsigned mates = 0xffffu << (tid & 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int x = 8; x > 0; x >>= 1) l[i] += __shfl_xor_sync(mates, l[i], x);
                int r = ty * 4 + i;
                if (r >= rows) continue;
                int token = w.first_token + (row0 + r) / share, head = w.kv_head * share + (row0 + r) % share;
                if (a.slots == 1) {
                    float inv = l[i] > 0.f ? 1.f / l[i] : l[i] == 0.f ? 0.f : l[i];      // (a NaN stays one)
                    T* to = static_cast<T*>(a.out) + (size_t)token * a.out_stride + (size_t)head * D;
#pragma unroll
                    for (int c = 0; c < COLS; ++c)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            if (c * 64 + tx * 4 + x < D) to[c * 64 + tx * 4 + x] = from_float<T>(o[i][c * 4 + x] * inv);
                } else {
                    size_t slot = ((size_t)token * a.n_heads + head) * a.slots + w.slot;
#pragma unroll
                    for (int c = 0; c < COLS; ++c)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            if (c * 64 + tx * 4 + x < D) a.acc[slot * D + c * 64 + tx * 4 + x] = o[i][c * 4 + x];
                    if (tx == 0) {
                        a.stats[slot * 2] = m[i];
                        a.stats[slot * 2 + 1] = l[i];
                    }
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ the parts joined
//
// A warp a row: each lane reads one part's maximum and sum, the weights are shared by shuffles, and the lanes take columns.
template <typename T>
__global__ void __launch_bounds__(128) prefix_attention_join_kernel(const __grid_constant__ Args a, int n_rows) {
    griddep_launch();
    griddep_wait();
    int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= n_rows) return;
    const int D = a.head_dim;
    const float* acc = behind_wait(a.acc) + (size_t)row * a.slots * D;
    const float* stats = behind_wait(a.stats) + (size_t)row * a.slots * 2;
    float m = -INFINITY;
    for (int s = lane; s < a.slots; s += 32) m = fmaxf(m, stats[s * 2]);
    m = warp_max(m);
    float against = m == -INFINITY ? 0.f : m, sum = 0.f;
    constexpr int COLS = LLMB_MAX_HEAD_DIM / 32;
    float value[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) value[c] = 0.f;
    for (int s0 = 0; s0 < a.slots; s0 += 32) {
        float weight = 0.f;
        if (s0 + lane < a.slots) {
            float l = stats[(s0 + lane) * 2 + 1];
            weight = l != 0.f ? exp2f(stats[(s0 + lane) * 2] - against) : 0.f;
            sum += l * weight;
        }
        int count = min(32, a.slots - s0);
        for (int s = 0; s < count; ++s) {
            float part = __shfl_sync(0xffffffffu, weight, s);
            if (part == 0.f) continue;                             // a part without keys has written no values
#pragma unroll
            for (int c = 0; c < COLS; ++c)
                if (c * 32 + lane < D) value[c] = fmaf(part, acc[(size_t)(s0 + s) * D + c * 32 + lane], value[c]);
        }
    }
    sum = warp_sum(sum);
    float inv = sum != 0.f ? 1.f / sum : 0.f;
    T* out = static_cast<T*>(a.out) + (size_t)(row / a.n_heads) * a.out_stride + (size_t)(row % a.n_heads) * D;
#pragma unroll
    for (int c = 0; c < COLS; ++c)
        if (c * 32 + lane < D) out[c * 32 + lane] = from_float<T>(value[c] * inv);
}

// ------------------------------------------------------------------------------------------------ the call

struct Plan {
    int prefix_tiles, prefix_splits, own_tiles, own_splits, slots;
};

constexpr int SMS = 148;

// Into how many parts the shared and the own pages are cut: as many pages a block as make all blocks come to about `wave`,
// two pages at least.
Plan plan_of(int n_seqs, int n_groups, int share, int n_kv_heads, int rows, int max_new, int max_group, int shared_pages, int own_pages, int wave) {
    Plan p;
    p.prefix_tiles = shared_pages > 0 ? ceil_div((long long)max_group * share, rows) : 0;
    p.own_tiles = ceil_div((long long)max_new * share, rows);
    long long prefix = (long long)n_groups * p.prefix_tiles * n_kv_heads, own = (long long)n_seqs * p.own_tiles * n_kv_heads;
    long long per = (prefix * shared_pages + own * own_pages + wave - 1) / wave;
    if (per < 2) per = 2;
    p.prefix_splits = shared_pages > 0 ? ceil_div(shared_pages, per) : 0;
    p.own_splits = ceil_div(own_pages, per);
    if (p.prefix_splits > 64) p.prefix_splits = 64;
    if (p.own_splits > 64) p.own_splits = 64;
    p.slots = p.prefix_splits + p.own_splits;
    return p;
}

// the least power of two that is no less than n: replayed steps of one bucket make the same launches
int bucket(int n) {
    int b = 1;
    while (b < n) b *= 2;
    return b;
}

Plan plan_for(int n_seqs, int n_groups, int n_heads, int n_kv_heads, int head_dim, int max_new, int max_group, int max_shared, int max_own) {
    int shared = max_shared > 0 ? bucket(max_shared) : 0, own = bucket(ceil_div(max_own > 0 ? max_own : 1, LLMB_PAGE));
    int an_sm = head_dim <= 64 ? 4 : head_dim <= 128 ? 2 : 1;
    return plan_of(n_seqs, n_groups, n_heads / n_kv_heads, n_kv_heads, SIMT_ROWS, max_new, max_group, shared, own, an_sm * SMS);
}

template <typename T, int DMAX>
int launch_simt(const Args& a, long long blocks, cudaStream_t stream) {
    constexpr size_t smem = simt_floats<DMAX>() * sizeof(float);
    static bool configured = false;
    if (!configured) {
        LLMB_CUDA(cudaFuncSetAttribute(prefix_attention_simt_kernel<T, DMAX>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        configured = true;
    }
    llmb::launch(prefix_attention_simt_kernel<T, DMAX>, dim3((unsigned)blocks), SIMT_THREADS, smem, stream, true, a);
    return check_launch("prefix_attention_simt");
}

template <typename T>
int run(const Args& a, int n_tokens, cudaStream_t stream) {
    long long blocks = (long long)a.n_kv_heads * ((long long)a.n_groups * a.prefix_tiles * a.prefix_splits + (long long)a.n_seqs * a.own_tiles * a.own_splits);
    LLMB_REQUIRE(blocks < (1ll << 31), "prefix_attention: too many blocks");
    int code = a.head_dim <= 64 ? launch_simt<T, 64>(a, blocks, stream)
             : a.head_dim <= 128 ? launch_simt<T, 128>(a, blocks, stream) : launch_simt<T, 256>(a, blocks, stream);
    if (code || a.slots == 1) return code;
    int rows = n_tokens * a.n_heads;
    llmb::launch(prefix_attention_join_kernel<T>, dim3((rows + 3) / 4), 128, 0, stream, true, a, rows);
    return check_launch("prefix_attention_join");
}

}  // namespace

// Floats of scratch that a call of these sizes needs, and the number of its launches in *kernels.
LLMB_EXPORT long long llmb_prefix_attention_scratch_floats(int n_tokens, int n_seqs, int n_groups, int n_heads, int n_kv_heads, int head_dim,
                                                           int max_new, int max_group, int max_shared, int max_own, int* kernels) {
    if (n_tokens <= 0 || n_seqs <= 0 || n_groups <= 0 || n_kv_heads <= 0 || n_heads < n_kv_heads) return 0;
    Plan p = plan_for(n_seqs, n_groups, n_heads, n_kv_heads, head_dim, max_new, max_group, max_shared, max_own);
    *kernels = p.slots > 1 ? 2 : 1;
    return p.slots > 1 ? (long long)n_tokens * n_heads * p.slots * (head_dim + 2) : 0;
}

LLMB_EXPORT int llmb_prefix_attention(const void* q, int q_stride, const void* k_cache, const void* v_cache, const int* block_table,
                                      int table_stride, const int* seq_lens, const int* cu_seqlens, const int* group_first,
                                      const int* group_pages, void* out, int out_stride, float* scratch, long long scratch_floats, int dtype,
                                      int n_tokens, int n_seqs, int n_groups, int n_heads, int n_kv_heads, int head_dim, float scale,
                                      int max_new, int max_group, int max_shared, int max_own, cudaStream_t stream) {
    if (n_tokens == 0 || n_seqs == 0) return LLMB_OK;
    LLMB_REQUIRE(n_tokens > 0 && n_seqs > 0 && n_groups > 0 && n_groups <= n_seqs, "prefix_attention: %d tokens of %d sequences in %d groups",
                 n_tokens, n_seqs, n_groups);
    LLMB_REQUIRE(n_kv_heads > 0 && n_heads % n_kv_heads == 0, "prefix_attention: %d heads are no multiple of %d kv heads", n_heads, n_kv_heads);
    LLMB_REQUIRE(head_dim > 0 && head_dim <= LLMB_MAX_HEAD_DIM, "prefix_attention: head_dim %d (served: up to %d)", head_dim, LLMB_MAX_HEAD_DIM);
    LLMB_REQUIRE(max_new > 0 && max_group >= max_new && max_shared >= 0 && max_own >= 0, "prefix_attention: bad sizes");
    LLMB_REQUIRE((long long)n_tokens * n_heads < (1ll << 31), "prefix_attention: %d tokens of %d heads", n_tokens, n_heads);
    Plan p = plan_for(n_seqs, n_groups, n_heads, n_kv_heads, head_dim, max_new, max_group, max_shared, max_own);
    long long rows = (long long)n_tokens * n_heads;
    LLMB_REQUIRE(p.slots == 1 || (scratch != nullptr && scratch_floats >= rows * p.slots * (head_dim + 2)), "prefix_attention: scratch too small");
    int size = dtype == LLMB_DTYPE_F32 ? 4 : 2;
    bool vectors = (head_dim * size) % 16 == 0 && ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) == 0;
    Args a{q, k_cache, v_cache, block_table, seq_lens, cu_seqlens, group_first, group_pages, out, scratch, scratch + rows * p.slots * head_dim,
           q_stride, out_stride, table_stride, n_seqs, n_groups, n_heads, n_kv_heads, head_dim, scale * LOG2E,
           p.prefix_tiles, p.prefix_splits, p.own_tiles, p.own_splits, p.slots, vectors ? 1 : 0};
    return dtype == LLMB_DTYPE_F32 ? run<float>(a, n_tokens, stream) : run<__nv_bfloat16>(a, n_tokens, stream);
}

// the packed doors of the launching entry points (common.cuh)
LLMB_PACKED(llmb_prefix_attention)
