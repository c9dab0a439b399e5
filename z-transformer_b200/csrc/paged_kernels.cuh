// A KV cache of pages: rows of keys and values in fixed-size pages of a pool that all sequences share, a table that names
// every sequence's pages in order, and the append of new rows.  (Their attention: decode_kernels.cuh for one new row a sequence,
// tc_rows.cuh for more.)
//
// Key slot j of sequence b is row j % page_size of page table[b, j / page_size]; a page's row holds n_kv_heads * dim
// floats.  New rows are ragged: sequence b has rows [cu_rows[b], cu_rows[b + 1]) of the new tensors (one each where
// cu_rows is null).  They are appended first and attend then, so the last of them stands at slot n_keys[b] - 1, and the
// query at position p sees slot j where j <= p and, with a window, where j > p - window or j < sinks.
//
// (The reference keeps a sequence's rows contiguous, src/kv_cache.zig:60-95, and appends one at a time.)
#pragma once

#include "zt_common.cuh"

namespace zt {

struct Pages {
    const float *k, *v;  // [n_pages, page_size, width]
    const int *table;    // [batch, max_pages]
    int n_pages, page_size, max_pages, width;
    uint32_t per;  // j / page_size is j * per >> shift for every j below 2^31
    int shift;
    // Elements from the pool's begin to the row of slot j of sequence b; negative where the table names no page for it.
    __device__ __forceinline__ long long row(int b, int j) const {
        return row_on(table[(long long)b * max_pages + page_of(j)], j);
    }
    // The same where the slot's page is known.
    __device__ __forceinline__ long long row_on(int id, int j) const {
        return id < 0 || id >= n_pages ? -1 : ((long long)id * page_size + (j - page_of(j) * page_size)) * width;
    }
    __device__ __forceinline__ int page_of(int j) const { return (int)(((uint64_t)(uint32_t)j * per) >> shift); }
    __device__ __forceinline__ long long capacity() const { return (long long)max_pages * page_size; }
};

// With L bits to hold page_size - 1 and `per` 2^(31 + L) / page_size rounded up, per page_size is at most 2^L over 2^(31 + L), so
// that j times the excess stays below one quotient's worth for 31 bits of j; `per` itself is below 2^32.
inline Pages make_pages(const float *k, const float *v, const int *table, int n_pages, int page_size, int max_pages, int width) {
    Pages p{k, v, table, n_pages, page_size, max_pages, width, 0, 31};
    while ((1LL << (p.shift - 31)) < page_size) ++p.shift;
    p.per = (uint32_t)(((1ull << p.shift) + (uint64_t)page_size - 1) / (uint64_t)page_size);
    return p;
}

// What a query at position p sees; `window` 0: everything up to itself.
struct Seen {
    int window, sinks;
    __device__ __forceinline__ bool operator()(int key, int pos) const { return key <= pos && (window == 0 || key > pos - window || key < sinks); }
};

// A sequence's new rows: [begin, begin + count) of `rows`, whose first stands at slot `pos`.
struct NewRows {
    int begin, count, pos;
    bool bad;  // the counts contradict each other or the tensors: nothing is read for such a sequence
};
// n_keys: the rows of the sequence with the new ones (`appended`), or before them.
__device__ __forceinline__ NewRows new_rows(const int *cu_rows, const int *n_keys, int b, int rows, const Pages &pg, bool appended) {
    NewRows r;
    r.begin = cu_rows ? cu_rows[b] : b;
    const int end = cu_rows ? cu_rows[b + 1] : b + 1, nk = n_keys[b];
    r.bad = r.begin < 0 || end < r.begin || end > rows;
    r.count = r.bad ? 0 : end - r.begin;
    r.pos = appended ? nk - r.count : nk;
    r.bad = r.bad || nk < 0 || r.pos < 0 || (long long)r.pos + r.count > pg.capacity();
    return r;
}

// The rows that sequence b answers for in an attention over pages, where a tile of 128 (row, head of a KV group) pairs belongs to one
// sequence: [begin, end), of which it computes those in front of `upto` and makes the rest NaN.  Where the bounds ascend they are its own.
// Elsewhere b answers from the greatest bound up to its own on (the first sequence from the least of all) to the greatest up to the
// next one, and those behind the least bound to come are other sequences' as well, or only a descent passes over them: so every
// row between the least and the greatest bound is one block's, and no row is computed that belongs to two sequences.
struct RowSpan {
    int b, begin, end, upto;  // b: -1 where the tile is nobody's
};
__host__ __device__ __forceinline__ int row_bound(const int *cu_rows, int rows, int i) {
    const int c = cu_rows[i];
    return c < 0 ? 0 : (c > rows ? rows : c);
}
// The first tile of a sequence that answers for rows from `begin` on: as many as it needs, or one more, lie in front of the next one's.
__host__ __device__ __forceinline__ long long first_row_tile(int begin, int group, int b) { return (long long)begin * group / 128 + b; }
// Whom tile `slot` belongs to, found one sequence after the other: for bounds that do not ascend.
__host__ __device__ inline RowSpan row_span(const int *cu_rows, int batch, int rows, int group, int slot) {
    RowSpan s{0, rows, 0, rows};
    for (int i = 0; i <= batch; ++i) {
        const int c = row_bound(cu_rows, rows, i);
        s.begin = c < s.begin ? c : s.begin;
    }
    s.end = row_bound(cu_rows, rows, 0);
    for (s.b = slot < first_row_tile(s.begin, group, 0) ? batch : 0; s.b < batch; ++s.b) {
        const int c = row_bound(cu_rows, rows, s.b + 1);
        s.end = c > s.end ? c : s.end;
        if (slot < first_row_tile(s.end, group, s.b + 1)) break;
        s.begin = s.end;
    }
    if (s.b == batch) return RowSpan{-1, 0, 0, 0};
    for (int i = s.b + 1; i <= batch; ++i) {
        const int c = row_bound(cu_rows, rows, i);
        s.upto = c < s.upto ? c : s.upto;
    }
    return s;
}

// ---- append ----------------------------------------------------------------------------------------------------------

struct AppendParams {
    Pages pg;
    float *k_pages, *v_pages;
    const float *k_new, *v_new;
    int *n_keys, *skipped;
    const int *cu_rows;
    int batch, rows;
};
// Whether all of a sequence's new rows have a place (called by whole blocks): none is written otherwise.
__device__ __forceinline__ bool rows_fit(const AppendParams &p, const NewRows &r, int b) {
    bool fits = !r.bad;
    if (fits && r.count > 0)
        for (int s = r.pos / p.pg.page_size + (int)threadIdx.x; s <= (r.pos + r.count - 1) / p.pg.page_size; s += (int)blockDim.x) {
            const int id = p.pg.table[(long long)b * p.pg.max_pages + s];
            if (id < 0 || id >= p.pg.n_pages) fits = false;
        }
    return __syncthreads_and(fits);
}
// The last of the first `batch` sequences that row `row` belongs to (-1: it belongs to none), and how many of them it belongs to: one, where
// the bounds ascend (called by whole blocks).
struct Owners {
    int last, n;
};
__device__ __forceinline__ Owners owners_of(const int *cu_rows, int batch, int row, Owners *found) {
    if (!cu_rows) return row < batch ? Owners{row, 1} : Owners{-1, 0};
    if (threadIdx.x == 0) *found = Owners{-1, 0};
    __syncthreads();
    for (int b = threadIdx.x; b < batch; b += blockDim.x)
        if (cu_rows[b] <= row && row < cu_rows[b + 1]) atomicMax(&found->last, b), atomicAdd(&found->n, 1);
    __syncthreads();
    return *found;
}

// A block per new row.  Where a sequence has one row only (cu_rows null) its block also advances the count; elsewhere rows of
// other blocks still read it, and advance_kernel follows.  A row in the bounds of several sequences, which do not ascend then, goes to
// each of them: their counts take it in.  2048 rows of 2 x 4 KB take 12.5 us, twice what their bytes take, the counts
// 6.6: what is waited for is a chain of dependent loads, the bounds, the count, the table, before the first byte is copied.
__global__ void __launch_bounds__(256) append_paged_kernel(const AppendParams p) {
    __shared__ Owners found;
    pdl_wait();
    pdl_launch();
    const int row = blockIdx.x;
    for (int below = p.batch, left = 1; left > 0;) {
        const Owners own = owners_of(p.cu_rows, below, row, &found);
        const int b = own.last;
        if (b < 0) return;
        const NewRows r = new_rows(p.cu_rows, p.n_keys, b, p.rows, p.pg, false);
        const bool fits = rows_fit(p, r, b);  // (behind its barrier everyone has read `found`)
        if (fits) {
            const long long at = p.pg.row(b, r.pos + (row - r.begin));
            const float *ks = p.k_new + (long long)row * p.pg.width, *vs = p.v_new + (long long)row * p.pg.width;
            float *kd = p.k_pages + at, *vd = p.v_pages + at;
            for (int j = threadIdx.x * 4; j < p.pg.width; j += 1024) {
                const float4 kx = *reinterpret_cast<const float4 *>(ks + j), vx = *reinterpret_cast<const float4 *>(vs + j);
                *reinterpret_cast<float4 *>(kd + j) = kx, *reinterpret_cast<float4 *>(vd + j) = vx;
            }
        }
        left = own.n - 1, below = b;
        if (p.cu_rows) continue;
        __syncthreads();  // (every thread has read the count)
        if (threadIdx.x == 0) {
            if (fits) p.n_keys[b] = r.pos + 1;
            else if (p.skipped) atomicAdd(p.skipped, 1);
        }
    }
}
// A block per sequence, behind append_paged_kernel: the counts take in the rows that it wrote.
__global__ void __launch_bounds__(128) advance_kernel(const AppendParams p) {
    pdl_wait();
    pdl_launch();
    const int b = blockIdx.x;
    const NewRows r = new_rows(p.cu_rows, p.n_keys, b, p.rows, p.pg, false);
    const bool fits = rows_fit(p, r, b);
    __syncthreads();
    if (threadIdx.x != 0) return;
    if (fits) p.n_keys[b] = r.pos + r.count;
    else if (p.skipped) atomicAdd(p.skipped, 1);
}
inline int launch_append_paged(const AppendParams &p, cudaStream_t stream) {
    if (p.rows > 0 && launch_pdl("append_paged_kernel", append_paged_kernel, dim3((unsigned)p.rows), dim3(256), 0, stream, p)) return 1;
    if (!p.cu_rows) return 0;
    return launch_pdl("advance_kernel", advance_kernel, dim3((unsigned)p.batch), dim3(128), 0, stream, p);
}

}  // namespace zt
