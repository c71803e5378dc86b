// Items of a pool copied to other places of the same pool, in every tensor at once: pages of a paged cache (all layers of keys and
// values in one tensor, or a tensor each), or the rows that recurrent layers keep for a sequence.
//
//   tensor[o, target_i, b, 0 .. rows_i - 1] = tensor[o, source_i, b, 0 .. rows_i - 1]     for every pair i, outer o, block b
//
// What forking a sequence needs (the last, partly filled page to a page of the child) and what compacting a pool needs (whole
// pages to lower places). There is no arithmetic: the bytes of every distinct source are read once and those of every target
// written once, and memory bounds it. Pairs are grouped by their source, so that a page that goes to sixteen places is read for
// one of them. No target is a source (the caller's promise, checked where the lists are made), so the order of blocks is free.
//
// * blockIdx = (slice of the run's bytes, run, tensor); a run is a source with its targets. A thread moves vectors of 16 bytes (8, 4
//   or 2 where an address, a stride or a row asks for less), MOVES of them in flight.
// * the lists travel as kernel arguments: nothing to allocate, to copy or to keep alive, and nothing a later call could overwrite.
#include "common.cuh"

using namespace llmb;

LLMB_DEFINE_LAST_ERROR(llmb_page_copy)

namespace {

constexpr int THREADS = 256;
constexpr int MOVES = 4;
constexpr int MAX_TENSORS = 16;       // of a launch
constexpr int MAX_PAIRS = 240;        // of a launch: the argument block stays below 4 KB

struct Tensor {
    unsigned char* base;
    long long outer_stride, item_stride, block_stride;      // bytes
    int outers, blocks;
    int row_vectors;                                        // of a row, in vectors
};
struct Copies {
    Tensor tensors[MAX_TENSORS];
    short run_first[MAX_PAIRS + 1];                         // the run's first pair
    int source[MAX_PAIRS];                                  // of a run
    int target[MAX_PAIRS];                                  // of a pair
    unsigned char rows[MAX_PAIRS];                          // of a pair, 1 .. 64
    unsigned char run_rows[MAX_PAIRS];                      // the most rows of a run's pairs
};
static_assert(sizeof(Copies) < 4000, "kernel arguments");

template <typename V>
__global__ void __launch_bounds__(THREADS) page_copy_kernel(const __grid_constant__ Copies c) {
    const Tensor& t = c.tensors[blockIdx.z];
    int run = blockIdx.y, first = c.run_first[run], last = c.run_first[run + 1];
    unsigned per_block = (unsigned)c.run_rows[run] * t.row_vectors;
    long long total = (long long)t.outers * t.blocks * per_block;
    long long at = (long long)blockIdx.x * (THREADS * MOVES) + threadIdx.x;
    if (at >= total) return;
    const unsigned char* from = t.base + (long long)c.source[run] * t.item_stride;
    V moved[MOVES];
    long long offset[MOVES];
    unsigned within[MOVES];
#pragma unroll
    for (int m = 0; m < MOVES; ++m) {
        long long i = at + m * THREADS;
        if (i < total) {
            long long strip = i / per_block;
            within[m] = (unsigned)(i - strip * per_block);
            int outer = (int)(strip / t.blocks), block = (int)(strip - (long long)outer * t.blocks);
            offset[m] = outer * t.outer_stride + block * t.block_stride + (long long)within[m] * sizeof(V);
            moved[m] = *reinterpret_cast<const V*>(from + offset[m]);
        } else {
            within[m] = 0xffffffffu;
        }
    }
    for (int pair = first; pair < last; ++pair) {
        unsigned char* to = t.base + (long long)c.target[pair] * t.item_stride;
        unsigned limit = (unsigned)c.rows[pair] * t.row_vectors;
#pragma unroll
        for (int m = 0; m < MOVES; ++m)
            if (within[m] < limit) *reinterpret_cast<V*>(to + offset[m]) = moved[m];
    }
}

}  // namespace

// n_tensors tensors, each described by 7 numbers in `shapes`: address, outers, blocks, then the strides of an outer, an item and a block and
// the size of a row, in bytes. n_pairs pairs (source, target, rows); equal sources must stand together. rows are 1 .. 64 rows of a block.
LLMB_EXPORT int llmb_page_copy(int n_tensors, const long long* shapes, int n_pairs, const int* pairs, cudaStream_t stream) {
    if (n_pairs == 0 || n_tensors == 0) return LLMB_OK;
    LLMB_REQUIRE(n_tensors > 0 && n_pairs > 0, "page_copy: bad sizes");
    for (int i = 0; i < n_pairs; ++i)
        LLMB_REQUIRE(pairs[3 * i] >= 0 && pairs[3 * i + 1] >= 0 && pairs[3 * i + 2] >= 1 && pairs[3 * i + 2] <= 64,
                     "page_copy: pair %d copies %d rows of %d to %d", i, pairs[3 * i + 2], pairs[3 * i], pairs[3 * i + 1]);
    for (int t0 = 0; t0 < n_tensors; t0 += MAX_TENSORS) {
        int count = n_tensors - t0 < MAX_TENSORS ? n_tensors - t0 : MAX_TENSORS;
        Copies c;
        unsigned long long bits = 0;
        long long widest = 0;                                    // bytes of one row over all strips of a tensor
        for (int t = 0; t < count; ++t) {
            const long long* s = shapes + 7 * (t0 + t);
            LLMB_REQUIRE(s[0] != 0 && s[1] > 0 && s[1] < (1ll << 31) && s[2] > 0 && s[2] < (1ll << 31) && s[6] > 0 && s[6] < (1ll << 31),
                         "page_copy: tensor %d is empty", t0 + t);
            c.tensors[t] = Tensor{reinterpret_cast<unsigned char*>(s[0]), s[3], s[4], s[5], (int)s[1], (int)s[2], (int)s[6]};
            bits |= (unsigned long long)s[0] | (unsigned long long)s[3] | (unsigned long long)s[4] | (unsigned long long)s[5] | (unsigned long long)s[6];
            long long row = s[1] * s[2] * s[6];
            if (row > widest) widest = row;
        }
        int vector = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
        LLMB_REQUIRE(bits % 2 == 0, "page_copy: elements of one byte");
        for (int t = 0; t < count; ++t) c.tensors[t].row_vectors /= vector;
        for (int p0 = 0; p0 < n_pairs; p0 += MAX_PAIRS) {
            int n = n_pairs - p0 < MAX_PAIRS ? n_pairs - p0 : MAX_PAIRS, runs = 0, most = 0;
            for (int i = 0; i < n; ++i) {
                const int* p = pairs + 3 * (p0 + i);
                if (i == 0 || p[0] != c.source[runs - 1]) {
                    c.source[runs] = p[0];
                    c.run_rows[runs] = 0;
                    c.run_first[runs++] = (short)i;
                }
                c.target[i] = p[1];
                c.rows[i] = (unsigned char)p[2];
                if (p[2] > c.run_rows[runs - 1]) c.run_rows[runs - 1] = (unsigned char)p[2];
                if (p[2] > most) most = p[2];
            }
            c.run_first[runs] = (short)n;
            long long slices = (widest / vector * most + THREADS * MOVES - 1) / (THREADS * MOVES);
            LLMB_REQUIRE(slices < (1ll << 31), "page_copy: a tensor of too many bytes");
            dim3 grid((unsigned)slices, runs, count);
            if (vector == 16) page_copy_kernel<uint4><<<grid, THREADS, 0, stream>>>(c);
            else if (vector == 8) page_copy_kernel<uint2><<<grid, THREADS, 0, stream>>>(c);
            else if (vector == 4) page_copy_kernel<unsigned><<<grid, THREADS, 0, stream>>>(c);
            else page_copy_kernel<unsigned short><<<grid, THREADS, 0, stream>>>(c);
            int code = check_launch("page_copy");
            if (code) return code;
        }
    }
    return LLMB_OK;
}
