// qdc_pages.hip -- the pages of a cache: rows that grow, fork, end and move together.
//
// Which page belongs to which row is kept on the device, so that a step needs no word
// from the host and can be captured.  The bookkeeping of a call is one workgroup's: it
// checks everything first (rows named twice by a bitmap in LDS) and then either does
// the whole call or none of it.  It is bound by the chain of dependent loads, rows ->
// lengths -> table -> refs, each a memory latency; the entries of a call are taken side
// by side and their pages as one flat list, a thread a page.  The copies are launches
// of their own that read what the first one decided.
#include "qdc_cache.hpp"

namespace qdc {
namespace {

constexpr int kBook = 1024;              // threads of the bookkeeping workgroup
constexpr int kBookWaves = kBook / kWave;
constexpr int kMaxRows = 1 << 18;        // rows of a cache: a bit each in LDS

struct Book {
    int32_t *table, *lengths, *refs, *free_pages;
    int64_t width;
    int n, rows, pages, shift;
    int32_t *error_flag;
};

// Agent scope: atomics are done in L2, past the first-level cache.
__device__ __forceinline__ int load_past_l1(const int32_t *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Everything this workgroup wrote or changed is seen by all of it.
__device__ __forceinline__ void settle() {
    __threadfence();
    __syncthreads();
}

// Exclusive prefix sum over the workgroup and the whole; `parts` is LDS scratch.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *parts, int64_t &all) {
    const int l = threadIdx.x % kWave, wv = threadIdx.x / kWave;
    int64_t inc = v;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int64_t o = __shfl_up(inc, d, kWave);
        if (l >= d) inc += o;
    }
    __syncthreads();  // the scratch is free
    if (l == kWave - 1) parts[wv] = inc;
    __syncthreads();
    int64_t before = 0;
    all = 0;
    for (int w = 0; w < kBookWaves; ++w) {
        const int64_t p = parts[w];
        if (w < wv) before += p;
        all += p;
    }
    return before + inc - v;
}

__device__ __forceinline__ void clear_bits(uint32_t *bits, int n) {
    for (int i = threadIdx.x; i < (n + 31) / 32; i += kBook) bits[i] = 0;
    __syncthreads();
}
__device__ __forceinline__ bool set_bit(uint32_t *bits, int i) {  // whether it was set
    return atomicOr(&bits[i >> 5], 1u << (i & 31)) >> (i & 31) & 1u;
}
__device__ __forceinline__ bool has_bit(const uint32_t *bits, int i) {
    return bits[i >> 5] >> (i & 31) & 1u;
}

__device__ __forceinline__ int64_t blocks_of(int64_t positions, int shift) {
    return (positions + ((int64_t)1 << shift) - 1) >> shift;
}

// The last entry whose run starts at or before `at`; starts[0] = 0, ascending.
__device__ __forceinline__ int run_of(const int64_t *starts, int n, int64_t at) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (starts[mid] <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A stack that may hold anything: the number of pages that can be taken from it.
__device__ __forceinline__ int64_t stack_count(const Book &b) {
    return min(max(b.free_pages[0], 0), b.pages);
}

__global__ __launch_bounds__(kBook) void pages_extend(Book b, int32_t *positions,
                                                      const int32_t *index,
                                                      const int32_t *counts) {
    extern __shared__ uint32_t seen[];
    __shared__ int64_t parts[kBookWaves], start[kBook];
    __shared__ int row_of[kBook], have_of[kBook];
    clear_bits(seen, b.rows);
    const int64_t count = stack_count(b), reach = b.width << b.shift;
    int64_t need = 0;
    bool bad = false;
    for (int i = threadIdx.x; i < b.n; i += kBook) {
        const int row = index[i];
        if (row < 0) continue;
        if (row >= b.rows || set_bit(seen, row)) {
            bad = true;
            continue;
        }
        const int64_t len = b.lengths[row], more = counts ? counts[i] : 1;
        bad = bad || len < 0 || more < 0 || len + more > reach;
        need += blocks_of(len + more, b.shift) - blocks_of(len, b.shift);
    }
    int64_t total;
    block_scan(need, parts, total);
    if (__syncthreads_or(bad || total > count)) {
        for (int i = threadIdx.x; i < b.n; i += kBook) positions[i] = -1;
        if (threadIdx.x == 0) raise_flag(b.error_flag);
        return;
    }
    int64_t taken = 0;  // pages of earlier chunks of entries
    for (int i0 = 0; i0 < b.n; i0 += kBook) {
        const int i = i0 + threadIdx.x, row = i < b.n ? index[i] : -1;
        int64_t pages = 0, have = 0, len = -1, more = 0;
        if (row >= 0) {
            len = b.lengths[row];
            more = counts ? counts[i] : 1;
            have = blocks_of(len, b.shift);
            pages = blocks_of(len + more, b.shift) - have;
            b.lengths[row] = (int32_t)(len + more);
        }
        if (i < b.n) positions[i] = (int32_t)len;
        int64_t all;
        start[threadIdx.x] = block_scan(pages, parts, all);
        row_of[threadIdx.x] = row;
        have_of[threadIdx.x] = (int)have;
        __syncthreads();
        for (int64_t p = threadIdx.x; p < all; p += kBook) {
            const int e = run_of(start, kBook, p);
            const int32_t page = b.free_pages[count - (taken + p)];
            b.table[row_of[e] * b.width + have_of[e] + (p - start[e])] = page;
            if ((uint32_t)page < (uint32_t)b.pages) b.refs[page] = 1;
        }
        taken += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) b.free_pages[0] = (int32_t)(count - total);
}

// Pages that the rows of a call list, flat: entry by entry, block by block.  A page is
// free when its refs, taken down once for each listing, reach nothing; the listing that
// puts it on the stack is its last, found by writing -(place + 1) over refs with a
// minimum.
__global__ __launch_bounds__(kBook) void pages_free(Book b, const int32_t *index) {
    extern __shared__ uint32_t seen[];
    __shared__ int64_t parts[kBookWaves], start[kBook];
    __shared__ int row_of[kBook];
    clear_bits(seen, b.rows);
    bool bad = false;
    for (int i = threadIdx.x; i < b.n; i += kBook) {
        const int row = index[i];
        if (row >= 0 && (row >= b.rows || set_bit(seen, row))) bad = true;
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) raise_flag(b.error_flag);
        return;
    }
    int64_t count = stack_count(b);
    // places of a chunk of entries in the flat list, those of its runs in LDS
    auto chunk = [&](int i0, int64_t &all) {
        const int i = i0 + threadIdx.x, row = i < b.n ? index[i] : -1;
        const int64_t len = row >= 0 ? b.lengths[row] : 0;
        const int64_t mine = min(max(blocks_of(len, b.shift), (int64_t)0), b.width);
        start[threadIdx.x] = block_scan(mine, parts, all);
        row_of[threadIdx.x] = row;
        __syncthreads();
    };
    auto entry = [&](int64_t p) {  // the table's place for place p of the chunk
        const int e = run_of(start, kBook, p);
        return row_of[e] * b.width + (p - start[e]);
    };
    int64_t before = 0, all = 0;
    int last = 0;
    for (int i0 = 0; i0 < b.n; i0 += kBook) {
        chunk(i0, all);
        for (int64_t p = threadIdx.x; p < all; p += kBook) {
            const int32_t page = b.table[entry(p)];
            if ((uint32_t)page < (uint32_t)b.pages) atomicSub(&b.refs[page], 1);
        }
        __syncthreads();
        last = i0;
        before += all;
    }
    settle();
    int64_t at = 0;
    for (int i0 = 0; i0 < b.n; i0 += kBook) {
        if (b.n > kBook) chunk(i0, all);
        for (int64_t p = threadIdx.x; p < all; p += kBook) {
            const int32_t page = b.table[entry(p)];
            if ((uint32_t)page < (uint32_t)b.pages && load_past_l1(&b.refs[page]) <= 0)
                atomicMin(&b.refs[page], -(int32_t)(at + p) - 1);
        }
        __syncthreads();
        at += all;
    }
    settle();
    // from the back: the first of the list ends on top
    for (int i0 = last; i0 >= 0; i0 -= kBook) {
        if (b.n > kBook) chunk(i0, all);
        before -= all;
        for (int64_t p0 = 0; p0 < all; p0 += kBook) {
            const int64_t p = all - 1 - (p0 + threadIdx.x);
            int32_t page = -1;
            int64_t place = 0;
            bool push = false;
            if (p >= 0) {
                place = entry(p);
                page = b.table[place];
                push = (uint32_t)page < (uint32_t)b.pages &&
                       load_past_l1(&b.refs[page]) == -(int32_t)(before + p) - 1;
            }
            int64_t pushed;
            const int64_t rank = block_scan(push, parts, pushed);
            if (push) {
                if (count + rank < b.pages) b.free_pages[1 + count + rank] = page;
                b.refs[page] = 0;
            }
            if (p >= 0) b.table[place] = -1;
            count += pushed;
        }
        __syncthreads();
        const int i = i0 + threadIdx.x;
        if (i < b.n && row_of[threadIdx.x] >= 0) b.lengths[row_of[threadIdx.x]] = 0;
        __syncthreads();
    }
    if (threadIdx.x == 0) b.free_pages[0] = (int32_t)min(count, (int64_t)b.pages);
}

// What the copies of a fork read: an entry's begun page, the new one, places used.
struct Copy {
    int32_t src, dst, used, pad;
};

__global__ __launch_bounds__(kBook) void pages_fork(Book b, const int32_t *parents,
                                                    const int32_t *children, Copy *copies) {
    extern __shared__ uint32_t seen[];
    __shared__ int64_t parts[kBookWaves], start[kBook];
    __shared__ int from[kBook], to[kBook];
    clear_bits(seen, b.rows);
    const int64_t count = stack_count(b);
    const int mask = (1 << b.shift) - 1;
    int64_t need = 0;
    bool bad = false;
    for (int i = threadIdx.x; i < b.n; i += kBook) {
        const int p = parents[i], c = children[i];
        if (p < 0 || c < 0) continue;
        if (p >= b.rows || c >= b.rows || set_bit(seen, c) || b.lengths[c] != 0) {
            bad = true;
            continue;
        }
        const int64_t len = b.lengths[p];
        bad = bad || len < 0 || blocks_of(len, b.shift) > b.width;
        need += (len & mask) != 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < b.n; i += kBook)
        if (parents[i] >= 0 && children[i] >= 0 && parents[i] < b.rows && has_bit(seen, parents[i]))
            bad = true;
    int64_t total;
    block_scan(need, parts, total);
    const bool refused = __syncthreads_or(bad || total > count);
    if (refused && threadIdx.x == 0) raise_flag(b.error_flag);
    int64_t taken = 0;
    for (int i0 = 0; i0 < b.n; i0 += kBook) {
        const int i = i0 + threadIdx.x;
        const int p = i < b.n ? parents[i] : -1, c = i < b.n ? children[i] : -1;
        const bool live = p >= 0 && c >= 0 && !refused;
        const int64_t len = live ? b.lengths[p] : 0;
        const int used = (int)(len & mask);
        int64_t all;
        const int64_t rank = block_scan(used != 0, parts, all);
        Copy copy = {-1, -1, 0, 0};
        if (live) {
            b.lengths[c] = (int32_t)len;
            if (used) {
                const int64_t at = len >> b.shift;
                copy.src = b.table[p * b.width + at];
                copy.dst = b.free_pages[count - (taken + rank)];
                copy.used = used;
                b.table[c * b.width + at] = copy.dst;
                if ((uint32_t)copy.dst < (uint32_t)b.pages) b.refs[copy.dst] = 1;
                if ((uint32_t)copy.src >= (uint32_t)b.pages ||
                    (uint32_t)copy.dst >= (uint32_t)b.pages) {
                    copy.used = 0;
                    raise_flag(b.error_flag);
                }
            }
        }
        if (i < b.n) copies[i] = copy;
        taken += all;
        start[threadIdx.x] = block_scan(len >> b.shift, parts, all);
        from[threadIdx.x] = p;
        to[threadIdx.x] = c;
        __syncthreads();
        for (int64_t k = threadIdx.x; k < all; k += kBook) {
            const int e = run_of(start, kBook, k);
            const int64_t j = k - start[e];
            const int32_t page = b.table[from[e] * b.width + j];
            b.table[to[e] * b.width + j] = page;
            if ((uint32_t)page < (uint32_t)b.pages) atomicAdd(&b.refs[page], 1);
        }
        __syncthreads();
    }
    if (threadIdx.x == 0 && !refused) b.free_pages[0] = (int32_t)(count - total);
}

// The used places of the begun pages: a workgroup per entry, plane and head.
__global__ __launch_bounds__(kBlock) void copy_begun(char *pool, const Copy *copies,
                                                     int64_t plane_bytes, int64_t page_bytes,
                                                     int heads, int64_t token_bytes) {
    const Copy c = copies[blockIdx.x];
    if (c.used == 0) return;
    const int plane = blockIdx.y / heads, head = blockIdx.y - plane * heads;
    char *base = pool + plane * plane_bytes + head * (page_bytes / heads);
    const u32x4 *src = reinterpret_cast<const u32x4 *>(base + c.src * page_bytes);
    u32x4 *dst = reinterpret_cast<u32x4 *>(base + c.dst * page_bytes);
    const int64_t chunks = c.used * token_bytes / 16;
    for (int64_t i = threadIdx.x; i < chunks; i += kBlock) dst[i] = src[i];
}

// Workspace of a move: count and pages in use, then the pages' new places, the holes
// and the pages that fill them.
struct Moves {
    int32_t *head, *place, *hole, *page;
};
__host__ __device__ inline Moves moves_in(void *workspace, int64_t pages) {
    int32_t *w = reinterpret_cast<int32_t *>(workspace);
    return Moves{w, w + 4, w + 4 + pages, w + 4 + 2 * pages};
}

__global__ __launch_bounds__(kBook) void pages_plan(int32_t *refs, int pages, Moves m) {
    __shared__ int64_t parts[kBookWaves];
    int64_t mine = 0, live, all;
    for (int i = threadIdx.x; i < pages; i += kBook) mine += refs[i] > 0;
    block_scan(mine, parts, live);
    int64_t holes = 0, movers = 0;
    for (int i0 = 0; i0 < pages; i0 += kBook) {
        const int i = i0 + threadIdx.x;
        const bool used = i < pages && refs[i] > 0;
        const bool hole = i < live && !used, mover = i >= live && used;
        const int64_t rank = block_scan(hole, parts, all);
        if (hole) m.hole[holes + rank] = i;
        holes += all;
        const int64_t rank2 = block_scan(mover, parts, all);
        if (mover) m.page[movers + rank2] = i;
        movers += all;
        if (i < pages) m.place[i] = i;
    }
    settle();
    for (int64_t k = threadIdx.x; k < movers; k += kBook) {
        const int page = m.page[k], hole = m.hole[k];
        m.place[page] = hole;
        refs[hole] = refs[page];
        refs[page] = 0;
    }
    if (threadIdx.x == 0) {
        m.head[0] = (int32_t)movers;
        m.head[1] = (int32_t)live;
    }
}

// The moves themselves, then the tables and the stack, spread over the grid.
__global__ __launch_bounds__(kBlock) void pages_move(char *pool, int64_t planes,
                                                     int64_t plane_bytes, int64_t page_bytes,
                                                     Moves m, int32_t *table, int64_t entries,
                                                     int32_t *free_pages, int pages) {
    const int count = m.head[0], live = m.head[1];
    for (int64_t u = blockIdx.x; u < count * planes; u += gridDim.x) {
        const int64_t k = u / planes, plane = u - k * planes;
        const u32x4 *src =
            reinterpret_cast<const u32x4 *>(pool + plane * plane_bytes + m.page[k] * page_bytes);
        u32x4 *dst = reinterpret_cast<u32x4 *>(pool + plane * plane_bytes + m.hole[k] * page_bytes);
        for (int64_t i = threadIdx.x; i < page_bytes / 16; i += kBlock) dst[i] = src[i];
    }
    const int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x, step = (int64_t)gridDim.x * kBlock;
    if (count)
        for (int64_t i = at; i < entries; i += step) {
            const int32_t page = table[i];
            if ((uint32_t)page < (uint32_t)pages) table[i] = m.place[page];
        }
    const int free_count = pages - live;
    for (int64_t i = at; i <= pages; i += step)
        free_pages[i] = i == 0 ? free_count : i <= free_count ? pages - (int)i : 0;
}

// A workgroup per pair and part of its bytes; each checks its own pair against the call.
__global__ __launch_bounds__(kBlock) void copy_items(char *pool, const int32_t *src,
                                                     const int32_t *dst, int n, int64_t planes,
                                                     int64_t plane_bytes, int items,
                                                     int64_t item_bytes, int32_t *error_flag) {
    const int i = blockIdx.x, s = src[i], d = dst[i];
    if (s < 0 || d < 0) return;
    bool bad = s >= items || d >= items;
    for (int j = threadIdx.x; j < n; j += kBlock) {
        const int sj = src[j], dj = dst[j];
        if (sj < 0 || dj < 0) continue;
        bad = bad || sj == d || (j < i && dj == d);
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) raise_flag(error_flag);
        return;
    }
    const int64_t chunks = item_bytes / 16;
    for (int64_t plane = 0; plane < planes; ++plane) {
        const u32x4 *from = reinterpret_cast<const u32x4 *>(pool + plane * plane_bytes + s * item_bytes);
        u32x4 *to = reinterpret_cast<u32x4 *>(pool + plane * plane_bytes + d * item_bytes);
        for (int64_t c = (int64_t)blockIdx.y * kBlock + threadIdx.x; c < chunks;
             c += (int64_t)gridDim.y * kBlock)
            to[c] = from[c];
    }
}

// The checks that all of these share.
int32_t check_book(const int32_t *table, const int32_t *lengths, const int32_t *refs,
                   const int32_t *free_pages, int64_t n, int64_t rows, int64_t width,
                   int64_t pages, int64_t page_size) {
    const int64_t lim = (int64_t)1 << 31;
    if (n < 0 || n >= ((int64_t)1 << 24) || rows <= 0 || rows >= kMaxRows || width <= 0 ||
        pages <= 0 || pages >= lim - 1 || page_shift(page_size) < 0 || width >= lim / page_size ||
        rows * width >= lim)
        return QDC_ERR_SHAPE;
    if (n && (!table || !lengths || !refs || !free_pages)) return QDC_ERR_NULL;
    return QDC_OK;
}

Book make_book(int32_t *table, int32_t *lengths, int32_t *refs, int32_t *free_pages, int64_t n,
               int64_t rows, int64_t width, int64_t pages, int64_t page_size,
               int32_t *error_flag) {
    return Book{table, lengths, refs, free_pages, width, (int)n, (int)rows, (int)pages,
                page_shift(page_size), error_flag};
}

// Bytes of a pool, -1 when they cannot be those of one allocation.
int64_t pool_bytes(int64_t planes, int64_t items, int64_t item_bytes) {
    const __int128 b = (__int128)planes * items * item_bytes;
    return b < ((__int128)1 << 48) ? (int64_t)b : -1;
}

uint32_t bit_bytes(int64_t rows) { return (uint32_t)(ceil_div(rows, (int64_t)32) * 4); }

}  // namespace
}  // namespace qdc

using namespace qdc;

#define QDC_BOOK_RANGES                                                                    \
    {table, rows * width * 4}, {lengths, rows * 4}, {refs, pages * 4},                     \
        {free_pages, (pages + 1) * 4}, {error_flag, error_flag ? 4 : 0}

extern "C" int32_t qdc_pages_extend(int32_t *positions, int32_t *table, int32_t *lengths,
                                    int32_t *refs, int32_t *free_pages, const int32_t *index,
                                    const int32_t *counts, int64_t n, int64_t rows, int64_t width,
                                    int64_t pages, int64_t page_size, int32_t *error_flag,
                                    hipStream_t stream) {
    const int32_t st = check_book(table, lengths, refs, free_pages, n, rows, width, pages, page_size);
    if (st != QDC_OK || n == 0) return st;
    if (!positions || !index) return QDC_ERR_NULL;
    const Range outs[6] = {{positions, n * 4}, QDC_BOOK_RANGES};
    const Range ins[2] = {{index, n * 4}, {counts, counts ? n * 4 : 0}};
    if (any_alias(outs, 6, ins, 2)) return QDC_ERR_ALIAS;
    hipLaunchKernelGGL(pages_extend, dim3(1), dim3(kBook), bit_bytes(rows), stream,
                       make_book(table, lengths, refs, free_pages, n, rows, width, pages, page_size,
                                 error_flag), positions, index, counts);
    return launch_status();
}

extern "C" int32_t qdc_pages_free(int32_t *table, int32_t *lengths, int32_t *refs,
                                  int32_t *free_pages, const int32_t *index, int64_t n,
                                  int64_t rows, int64_t width, int64_t pages, int64_t page_size,
                                  int32_t *error_flag, hipStream_t stream) {
    const int32_t st = check_book(table, lengths, refs, free_pages, n, rows, width, pages, page_size);
    if (st != QDC_OK || n == 0) return st;
    if (!index) return QDC_ERR_NULL;
    const Range outs[5] = {QDC_BOOK_RANGES};
    const Range ins[1] = {{index, n * 4}};
    if (any_alias(outs, 5, ins, 1)) return QDC_ERR_ALIAS;
    hipLaunchKernelGGL(pages_free, dim3(1), dim3(kBook), bit_bytes(rows), stream,
                       make_book(table, lengths, refs, free_pages, n, rows, width, pages, page_size,
                                 error_flag), index);
    return launch_status();
}

extern "C" int32_t qdc_pages_fork(int32_t *table, int32_t *lengths, int32_t *refs,
                                  int32_t *free_pages, const int32_t *parents,
                                  const int32_t *children, int64_t n, int64_t rows, int64_t width,
                                  int64_t pages, int64_t page_size, void *pool, int64_t planes,
                                  int64_t heads, int64_t token_bytes, void *workspace,
                                  int64_t workspace_bytes, int32_t *error_flag,
                                  hipStream_t stream) {
    const int32_t st = check_book(table, lengths, refs, free_pages, n, rows, width, pages, page_size);
    if (st != QDC_OK) return st;
    // a workgroup per entry, plane and head in a grid of fewer than 2^32 work-items
    if (planes < 0 ||
        (planes > 0 && (heads <= 0 || token_bytes <= 0 || token_bytes % 16 || planes >= 65536 ||
                        heads >= 65536 || planes * heads >= 65536 || token_bytes >= (1 << 24) ||
                        n * planes * heads >= (1 << 24))))
        return QDC_ERR_SHAPE;
    const int64_t page_bytes = planes ? heads * page_size * token_bytes : 0;
    const int64_t bytes = pool_bytes(planes, pages, page_bytes);
    if (bytes < 0) return QDC_ERR_SHAPE;
    if (n == 0) return QDC_OK;
    if (!parents || !children || !workspace || (planes > 0 && !pool)) return QDC_ERR_NULL;
    if (workspace_bytes < 16 * n || !aligned16(workspace) || !aligned16(pool)) return QDC_ERR_SHAPE;
    const Range outs[7] = {QDC_BOOK_RANGES, {workspace, 16 * n}, {pool, bytes}};
    const Range ins[2] = {{parents, n * 4}, {children, n * 4}};
    if (any_alias(outs, 7, ins, 2)) return QDC_ERR_ALIAS;
    Copy *copies = reinterpret_cast<Copy *>(workspace);
    hipLaunchKernelGGL(pages_fork, dim3(1), dim3(kBook), bit_bytes(rows), stream,
                       make_book(table, lengths, refs, free_pages, n, rows, width, pages, page_size,
                                 error_flag), parents, children, copies);
    const int32_t status = launch_status();
    if (status != QDC_OK || planes == 0) return status;
    hipLaunchKernelGGL(copy_begun, dim3((uint32_t)n, (uint32_t)(planes * heads)), dim3(kBlock), 0,
                       stream, (char *)pool, copies, pages * page_bytes, page_bytes, (int)heads,
                       token_bytes);
    return launch_status();
}

extern "C" int64_t qdc_pages_compact_workspace(int64_t pages) {
    return pages <= 0 || pages >= ((int64_t)1 << 31) - 1 ? 0 : 16 + 12 * pages;
}

extern "C" int32_t qdc_pages_compact(int32_t *table, int32_t *refs, int32_t *free_pages,
                                     int64_t rows, int64_t width, int64_t pages, void *pool,
                                     int64_t planes, int64_t page_bytes, void *workspace,
                                     int64_t workspace_bytes, hipStream_t stream) {
    const int64_t need = qdc_pages_compact_workspace(pages), lim = (int64_t)1 << 31;
    if (need == 0 || rows <= 0 || width <= 0 || rows >= lim || width >= lim || rows * width >= lim ||
        planes < 0 || planes >= 65536 ||
        (planes > 0 && (page_bytes <= 0 || page_bytes % 16 || page_bytes >= lim)))
        return QDC_ERR_SHAPE;
    const int64_t bytes = planes ? pool_bytes(planes, pages, page_bytes) : 0;
    if (bytes < 0) return QDC_ERR_SHAPE;
    if (!table || !refs || !free_pages || !workspace || (planes > 0 && !pool)) return QDC_ERR_NULL;
    if (workspace_bytes < need || !aligned16(workspace) || !aligned16(pool)) return QDC_ERR_SHAPE;
    const Range outs[5] = {{table, rows * width * 4}, {refs, pages * 4},
                           {free_pages, (pages + 1) * 4}, {workspace, need},
                           {pool, bytes}};
    if (any_alias(outs, 5, outs, 0)) return QDC_ERR_ALIAS;
    const Moves m = moves_in(workspace, pages);
    hipLaunchKernelGGL(pages_plan, dim3(1), dim3(kBook), 0, stream, refs, (int)pages, m);
    const int32_t status = launch_status();
    if (status != QDC_OK) return status;
    hipLaunchKernelGGL(pages_move, dim3(2048), dim3(kBlock), 0, stream, (char *)pool, planes,
                       pages * page_bytes, page_bytes, m, table, rows * width, free_pages,
                       (int)pages);
    return launch_status();
}

extern "C" int32_t qdc_copy_pages(void *pool, const int32_t *src, const int32_t *dst, int64_t n,
                                  int64_t planes, int64_t items, int64_t item_bytes,
                                  int32_t *error_flag, hipStream_t stream) {
    const int64_t lim = (int64_t)1 << 31;
    if (n < 0 || n >= ((int64_t)1 << 16) || planes < 0 || planes >= lim || items <= 0 ||
        items >= lim || item_bytes < 0 || item_bytes % 16 || item_bytes >= ((int64_t)1 << 40))
        return QDC_ERR_SHAPE;
    const int64_t bytes = pool_bytes(planes, items, item_bytes);
    if (bytes < 0) return QDC_ERR_SHAPE;
    if (n == 0 || planes == 0 || item_bytes == 0) return QDC_OK;
    if (!pool || !src || !dst) return QDC_ERR_NULL;
    if (!aligned16(pool)) return QDC_ERR_SHAPE;
    const Range outs[2] = {{pool, bytes}, {error_flag, error_flag ? 4 : 0}};
    const Range ins[2] = {{src, n * 4}, {dst, n * 4}};
    if (any_alias(outs, 2, ins, 2)) return QDC_ERR_ALIAS;
    hipLaunchKernelGGL(copy_items, dim3((uint32_t)n, 16), dim3(kBlock), 0, stream, (char *)pool,
                       src, dst, (int)n, planes, items * item_bytes, (int)items, item_bytes,
                       error_flag);
    return launch_status();
}
