// qdc_pages.hip -- the pages of a cache: rows that grow, fork, end and move together.
//
// Which page belongs to which row is kept on the device, so that a step needs no word
// from the host and can be captured.  The bookkeeping of a call is one workgroup's: it
// checks everything first (rows named twice by a bitmap in LDS) and then either does
// the whole call or none of it.  It is bound by the chain of dependent loads, rows ->
// lengths -> table -> refs, each a memory latency; the entries of a call are taken side
// by side, a thread an entry, whose values stay in registers from the checks to the
// work (past kBook entries they are read again), and their pages as one flat list, a
// thread a page: 5 to 8 us a call, of which a launch alone is 2.  The copies are bound by
// memory and are launches of their own that read what the first one decided.
#include "qdc_cache.hpp"

namespace qdc {
namespace {

constexpr int kBook = 1024;              // threads of the bookkeeping workgroup
constexpr int kBookWaves = kBook / kWave;
constexpr int kMaxRows = 1 << 18;        // rows of a cache: a bit each in LDS
// pages, and places of a table: lists of them are walked in steps of kBook, in 32 bits
constexpr int64_t kMaxPages = ((int64_t)1 << 31) - kBook;

struct Book {
    int32_t *table, *lengths, *refs, *free_pages;
    int64_t width;
    int n, rows, pages, shift;
    int32_t *error_flag;
};

// refs are counted with atomics, done in L2: a load of them goes past the first-level
// cache, and a barrier follows the atomics' returned values.
__device__ __forceinline__ int load_past_l1(const int32_t *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Exclusive prefix sum over the workgroup and the whole; `parts` is LDS scratch.
__device__ __forceinline__ int block_scan(int v, int *parts, int &all) {
    static_assert(kBookWaves == 16, "a row of lanes");
    const int l = threadIdx.x % kWave, wv = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int inc = wave_scan(v);
    __syncthreads();  // the scratch is free
    if (l == kWave - 1) parts[wv] = inc;
    __syncthreads();
    const int ends = row_scan(parts[l % kBookWaves]);
    all = __builtin_amdgcn_readlane(ends, kBookWaves - 1);
    return (wv ? __builtin_amdgcn_readlane(ends, wv - 1) : 0) + inc - v;
}

// Whether any thread says so, with the sum of v (below 2^31) over all of them.
__device__ __forceinline__ bool block_sum_or(int v, bool any, int *parts, int &all) {
    const bool some = __syncthreads_or(any);
    block_scan(some ? 0 : v, parts, all);
    return some;
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

__device__ __forceinline__ int blocks_of(int64_t positions, int shift) {
    return (int)((positions + ((int64_t)1 << shift) - 1) >> shift);
}

// The last entry whose run starts at or before `at`; starts[0] = 0, ascending.
__device__ __forceinline__ int run_of(const int *starts, int n, int at) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (starts[mid] <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A stack that may hold anything: the number of pages that can be taken from it.
__device__ __forceinline__ int stack_count(const Book &b) {
    return min(max(b.free_pages[0], 0), b.pages);
}

// An entry that grows: its row, length, and the pages it has and needs.
struct Growth {
    int row, len, more, have, need;
    bool bad;
};
__device__ __forceinline__ Growth growth_of(const Book &b, const int32_t *index,
                                            const int32_t *counts, int i) {
    Growth g = {-1, -1, 0, 0, 0, false};
    if (i >= b.n) return g;
    const int row = index[i], more = counts ? counts[i] : 1;
    if (row < 0) return g;
    g.bad = row >= b.rows;
    if (g.bad) return g;
    const int len = b.lengths[row];
    g.bad = len < 0 || more < 0 || (int64_t)len + more > b.width << b.shift;
    if (g.bad) return g;
    g.row = row;
    g.len = len;
    g.more = more;
    g.have = blocks_of(len, b.shift);
    g.need = blocks_of((int64_t)len + more, b.shift) - g.have;
    return g;
}

__global__ __launch_bounds__(kBook) void pages_extend(Book b, int32_t *positions,
                                                      const int32_t *index,
                                                      const int32_t *counts) {
    extern __shared__ uint32_t seen[];
    __shared__ int parts[kBookWaves], start[kBook], row_of[kBook], have_of[kBook];
    const int count = stack_count(b);
    const Growth mine = growth_of(b, index, counts, threadIdx.x);
    clear_bits(seen, b.rows);
    int need = mine.need;
    bool bad = mine.bad || (mine.row >= 0 && set_bit(seen, mine.row));
    for (int i = threadIdx.x + kBook; i < b.n; i += kBook) {
        const Growth g = growth_of(b, index, counts, i);
        bad = bad || g.bad || (g.row >= 0 && set_bit(seen, g.row));
        need += g.need;
    }
    int total;  // distinct rows: at most rows * width, below 2^31
    bad = block_sum_or(need, bad, parts, total);
    if (bad || total > count) {
        for (int i = threadIdx.x; i < b.n; i += kBook) positions[i] = -1;
        if (threadIdx.x == 0) raise_flag(b.error_flag);
        return;
    }
    int taken = 0;  // pages of earlier chunks of entries
    for (int i0 = 0; i0 < b.n; i0 += kBook) {
        const int i = i0 + threadIdx.x;
        const Growth g = i0 ? growth_of(b, index, counts, i) : mine;
        if (i < b.n) positions[i] = g.len;
        if (g.row >= 0) b.lengths[g.row] = g.len + g.more;
        if (total == 0) continue;
        int all;
        start[threadIdx.x] = block_scan(g.need, parts, all);
        row_of[threadIdx.x] = g.row;
        have_of[threadIdx.x] = g.have;
        __syncthreads();
        for (int p = threadIdx.x; p < all; p += kBook) {
            const int e = run_of(start, kBook, p);
            const int32_t page = b.free_pages[count - (taken + p)];
            b.table[row_of[e] * b.width + have_of[e] + (p - start[e])] = page;
            if ((uint32_t)page < (uint32_t)b.pages) b.refs[page] = 1;
        }
        taken += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) b.free_pages[0] = count - total;
}

// Pages that the rows of a call list, flat: entry by entry, block by block.  A page is
// free when its refs, taken down once for each listing, reach nothing.  The listing
// that takes down the last is the only one unless another took down before it; where
// that happened to a page that is now free, the listing that puts it on the stack is
// its last, found by writing -(place + 1) over refs with a minimum.
__global__ __launch_bounds__(kBook) void pages_free(Book b, const int32_t *index) {
    extern __shared__ uint32_t seen[];
    __shared__ int parts[kBookWaves], start[kBook], row_of[kBook];
    int count = stack_count(b);
    const int first = threadIdx.x < b.n ? index[threadIdx.x] : -1;
    const int first_len = first >= 0 && first < b.rows ? b.lengths[first] : 0;
    clear_bits(seen, b.rows);
    bool bad = first >= b.rows || (first >= 0 && set_bit(seen, first));
    for (int i = threadIdx.x + kBook; i < b.n; i += kBook) {
        const int row = index[i];
        bad = bad || row >= b.rows || (row >= 0 && set_bit(seen, row));
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) raise_flag(b.error_flag);
        return;
    }
    // a chunk of entries: the places of its runs in the flat list, and how many
    auto chunk = [&](int i0) {
        const int i = i0 + threadIdx.x;
        const int row = i0 == 0 ? first : i < b.n ? index[i] : -1;
        const int len = i0 == 0 ? first_len : row >= 0 ? b.lengths[row] : 0;
        int all;
        start[threadIdx.x] =
            block_scan((int)min((int64_t)blocks_of(max(len, 0), b.shift), b.width), parts, all);
        row_of[threadIdx.x] = row;
        __syncthreads();
        return all;
    };
    auto entry = [&](int p) {  // the table's place for place p of the chunk
        const int e = run_of(start, kBook, p);
        return row_of[e] * b.width + (p - start[e]);
    };
    // one chunk whose pages are a thread's each: they stay in registers
    int before = 0, all = chunk(0);
    const bool small = b.n <= kBook && all <= kBook;
    int64_t place = -1;
    int32_t page = -1;
    bool alone = false;  // this listing took down the last
    bool shared = false; // a page that several listed may be free
    for (int i0 = 0;;) {
        for (int p = threadIdx.x; p < all; p += kBook) {
            place = entry(p);
            page = b.table[place];
            if ((uint32_t)page >= (uint32_t)b.pages) continue;
            const int old = atomicSub(&b.refs[page], 1);
            alone = old <= 1;
            shared = shared || old > 1;
        }
        before += all;
        i0 += kBook;
        if (i0 >= b.n) break;
        __syncthreads();
        all = chunk(i0);
    }
    // (when not small, any page that others hold too asks for the second pass)
    bool second = __syncthreads_or(shared);
    if (second && small)
        second = __syncthreads_or(shared && load_past_l1(&b.refs[page]) <= 0);
    const int chunks = (b.n + kBook - 1) / kBook;
    if (second || !small) {
        int at = 0, seen_min = 0;
        for (int c = 0; c < chunks; ++c) {
            if (chunks > 1) {
                __syncthreads();
                all = chunk(c * kBook);
            }
            for (int p = threadIdx.x; p < all; p += kBook) {
                const int32_t q = b.table[entry(p)];
                if ((uint32_t)q < (uint32_t)b.pages && load_past_l1(&b.refs[q]) <= 0)
                    seen_min |= atomicMin(&b.refs[q], -(at + p) - 1);
            }
            at += all;
        }
        asm volatile("" ::"v"(seen_min));  // waited for
        __syncthreads();
    }
    // from the back: the first of the list ends on top
    for (int c = chunks - 1; c >= 0; --c) {
        if (chunks > 1) {
            __syncthreads();
            all = chunk(c * kBook);
        }
        before -= all;
        for (int p0 = 0; p0 < all; p0 += kBook) {
            const int p = all - 1 - (p0 + (int)threadIdx.x);
            bool push = false;
            int64_t where = -1;
            int32_t q = -1;
            if (small) {  // thread t holds place t: hand it to the one that counts from the back
                where = place;
                q = page;
                push = (uint32_t)q < (uint32_t)b.pages &&
                       (second ? load_past_l1(&b.refs[q]) == -(int)threadIdx.x - 1 : alone);
            } else if (p >= 0) {
                where = entry(p);
                q = b.table[where];
                push = (uint32_t)q < (uint32_t)b.pages &&
                       load_past_l1(&b.refs[q]) == -(before + p) - 1;
            }
            int pushed;
            int rank = block_scan(push, parts, pushed);
            if (small) rank = pushed - 1 - rank;
            if (push) {
                if (count + rank < b.pages) b.free_pages[1 + count + rank] = q;
                b.refs[q] = 0;
            }
            if (where >= 0) b.table[where] = -1;
            count += pushed;
        }
        const int i = c * kBook + threadIdx.x;
        if (i < b.n && row_of[threadIdx.x] >= 0) b.lengths[row_of[threadIdx.x]] = 0;
    }
    if (threadIdx.x == 0) b.free_pages[0] = min(count, b.pages);
}

// What the copies of a fork read: an entry's begun page, the new one, places used.
struct Copy {
    int32_t src, dst, used, pad;
};

// A pair that forks: -1 rows when it is left out.
struct Pair {
    int parent, child, len;
    bool bad;
};
__device__ __forceinline__ Pair pair_of(const Book &b, const int32_t *parents,
                                        const int32_t *children, int i) {
    Pair f = {-1, -1, 0, false};
    if (i >= b.n) return f;
    const int p = parents[i], c = children[i];
    if (p < 0 || c < 0) return f;
    f.bad = p >= b.rows || c >= b.rows;
    if (f.bad) return f;
    f.parent = p;
    f.child = c;
    f.len = b.lengths[p];
    f.bad = b.lengths[c] != 0 || f.len < 0 || blocks_of(f.len, b.shift) > b.width;
    return f;
}

// A pool whose begun pages are copied: `planes` planes of [pages, heads, page_size] rows.
struct Pool {
    char *data;
    int64_t plane_bytes, page_bytes, token_bytes;
    int planes, heads;
};

// `copies` NULL: this workgroup copies the begun pages itself (one chunk of entries).
__global__ __launch_bounds__(kBook) void pages_fork(Book b, const int32_t *parents,
                                                    const int32_t *children, Copy *copies,
                                                    Pool pool) {
    extern __shared__ uint32_t seen[];
    __shared__ int parts[kBookWaves], start[kBook], from[kBook], to[kBook];
    __shared__ Copy own[kBook];
    const int count = stack_count(b), mask = (1 << b.shift) - 1;
    const Pair mine = pair_of(b, parents, children, threadIdx.x);
    clear_bits(seen, b.rows);
    int need = (mine.len & mask) != 0;
    bool bad = mine.bad || (mine.child >= 0 && set_bit(seen, mine.child));
    for (int i = threadIdx.x + kBook; i < b.n; i += kBook) {
        const Pair f = pair_of(b, parents, children, i);
        bad = bad || f.bad || (f.child >= 0 && set_bit(seen, f.child));
        need += (f.len & mask) != 0;
    }
    __syncthreads();  // all children are marked: no parent may be one
    bad = bad || (mine.parent >= 0 && has_bit(seen, mine.parent));
    for (int i = threadIdx.x + kBook; i < b.n; i += kBook) {
        const int p = parents[i];
        bad = bad || (children[i] >= 0 && p >= 0 && p < b.rows && has_bit(seen, p));
    }
    int total;
    bad = block_sum_or(need, bad, parts, total);
    const bool refused = bad || total > count;
    if (refused && threadIdx.x == 0) raise_flag(b.error_flag);
    int taken = 0;
    for (int i0 = 0; i0 < b.n; i0 += kBook) {
        const int i = i0 + threadIdx.x;
        const Pair f = i0 ? pair_of(b, parents, children, i) : mine;
        const bool live = f.parent >= 0 && !refused;
        const int len = live ? f.len : 0, used = len & mask;
        int all;
        const int rank = block_scan(used != 0, parts, all);
        Copy copy = {-1, -1, 0, 0};
        if (live) b.lengths[f.child] = len;
        if (used) {
            const int at = len >> b.shift;
            copy.src = b.table[f.parent * b.width + at];
            copy.dst = b.free_pages[count - (taken + rank)];
            copy.used = used;
            b.table[f.child * b.width + at] = copy.dst;
            if ((uint32_t)copy.dst < (uint32_t)b.pages) b.refs[copy.dst] = 1;
            if ((uint32_t)copy.src >= (uint32_t)b.pages || (uint32_t)copy.dst >= (uint32_t)b.pages) {
                copy.used = 0;
                raise_flag(b.error_flag);
            }
        }
        if (!copies) own[threadIdx.x] = copy;
        else if (i < b.n) copies[i] = copy;
        taken += all;
        if (refused) continue;
        start[threadIdx.x] = block_scan(len >> b.shift, parts, all);
        from[threadIdx.x] = f.parent;
        to[threadIdx.x] = f.child;
        __syncthreads();
        for (int k = threadIdx.x; k < all; k += kBook) {
            const int e = run_of(start, kBook, k), j = k - start[e];
            const int32_t page = b.table[from[e] * b.width + j];
            b.table[to[e] * b.width + j] = page;
            if ((uint32_t)page < (uint32_t)b.pages) atomicAdd(&b.refs[page], 1);
        }
        __syncthreads();
    }
    if (threadIdx.x == 0 && !refused) b.free_pages[0] = count - total;
    if (copies || refused) return;
    const int per = pool.planes * pool.heads, l = threadIdx.x % kWave;  // a wavefront each
    for (int u = threadIdx.x / kWave; u < b.n * per; u += kBookWaves) {
        const Copy c = own[u / per];
        const int plane = u % per / pool.heads, head = u % per % pool.heads;
        char *base = pool.data + plane * pool.plane_bytes + head * (pool.page_bytes / pool.heads);
        const u32x4 *src = reinterpret_cast<const u32x4 *>(base + c.src * pool.page_bytes);
        u32x4 *dst = reinterpret_cast<u32x4 *>(base + c.dst * pool.page_bytes);
        for (int k = l; k < c.used * pool.token_bytes / 16; k += kWave) dst[k] = src[k];
    }
}

// A workgroup's copy of `chunks` 16-byte chunks: up to four loads a thread ahead of their
// stores, the stores as a stream.
__device__ __forceinline__ void copy_chunks(const char *src, char *dst, int64_t chunks) {
    constexpr int U = 4;
    const u32x4 *from = reinterpret_cast<const u32x4 *>(src);
    const int step = blockDim.x;
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * step < chunks; i += U * step) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load_raw(from + i + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) store_raw(dst + 16 * (i + u * step), v[u]);
    }
    for (; i < chunks; i += step) store_raw(dst + 16 * i, load_raw(from + i));
}

// The used places of the begun pages: a workgroup per entry, plane, head and piece.
constexpr int64_t kBegun = 8192;

__global__ __launch_bounds__(kBlock) void copy_begun(Pool pool, const Copy *copies) {
    const Copy c = copies[blockIdx.x];
    const int64_t at = blockIdx.z * kBegun, bytes = c.used * pool.token_bytes;
    if (at >= bytes) return;
    const int plane = blockIdx.y / pool.heads, head = blockIdx.y - plane * pool.heads;
    char *base =
        pool.data + plane * pool.plane_bytes + head * (pool.page_bytes / pool.heads) + at;
    copy_chunks(base + c.src * pool.page_bytes, base + c.dst * pool.page_bytes,
                min(kBegun, bytes - at) / 16);
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
    __shared__ int parts[kBookWaves];
    int mine = 0, live, all;
    for (int i = threadIdx.x; i < pages; i += kBook) mine += refs[i] > 0;
    block_scan(mine, parts, live);
    int holes = 0, movers = 0;
    for (int i0 = 0; i0 < pages; i0 += kBook) {
        const int i = i0 + threadIdx.x;
        const bool used = i < pages && refs[i] > 0;
        // pages below `live` are holes or stay, the others move or stay free
        const bool hole = i < live && !used, mover = i >= live && used;
        const int both = block_scan((int)hole | (int)mover << 16, parts, all);
        if (hole) m.hole[holes + (both & 0xffff)] = i;
        if (mover) m.page[movers + (both >> 16)] = i;
        if (i < pages) m.place[i] = i;
        holes += all & 0xffff;
        movers += all >> 16;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += kBook) {
        const int page = m.page[k], hole = m.hole[k];
        m.place[page] = hole;
        refs[hole] = refs[page];
        refs[page] = 0;
    }
    if (threadIdx.x == 0) {
        m.head[0] = movers;
        m.head[1] = live;
    }
}

// The moves themselves, a workgroup a piece of a page at a time, plane after plane, then
// the tables and the stack, spread over the grid.  Small pieces side by side keep what is
// copied at one time close together: 2 x 215 MB of pages of 64 KB in 12 planes 69 us (6.2
// TB/s), page after page 76, in pieces of 16 KB 76; with plain loads 72, plain stores 80.
constexpr int64_t kPiece = 4096;
constexpr uint32_t kMoveGrid = 16384;

__global__ __launch_bounds__(kBlock) void pages_move(char *pool, int64_t planes,
                                                     int64_t plane_bytes, int64_t page_bytes,
                                                     Moves m, int32_t *table, int64_t entries,
                                                     int32_t *free_pages, int pages) {
    const int count = m.head[0], live = m.head[1];
    const int64_t pieces = (page_bytes + kPiece - 1) / kPiece, per_plane = count * pieces;
    for (int64_t u = blockIdx.x; u < planes * per_plane; u += gridDim.x) {
        const int64_t plane = u / per_plane, rest = u - plane * per_plane;
        const int64_t k = rest / pieces, at = (rest - k * pieces) * kPiece;
        char *base = pool + plane * plane_bytes + at;
        const char *from = base + m.page[k] * page_bytes;
        char *to = base + m.hole[k] * page_bytes;
        const int chunks = (int)(min(kPiece, page_bytes - at) / 16);
        for (int i = threadIdx.x; i < chunks; i += kBlock)
            store_raw(to + 16 * i, load_stream(from + 16 * i));
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

// A workgroup per pair and part of a plane's item; each checks the call's pairs for itself.
// 8 rows' states of 19 MB to 5 places each (151 MB read, 755 MB written): 150 us = 6.0 TB/s
// in parts of 64 KB by 1024 threads; 165 in parts of 32 KB, 174 of 16 KB by 256, and 158 to
// 172 with two to five pairs of one src in a workgroup, which reads them once: the reads of
// the other pairs come from the caches as it is.
constexpr int kPart = 1024;

__global__ __launch_bounds__(kPart) void copy_items(char *pool, const int32_t *src,
                                                    const int32_t *dst, int n,
                                                    int64_t plane_bytes, int items,
                                                    int64_t item_bytes, int64_t part_bytes,
                                                    int parts, int32_t *error_flag) {
    __shared__ int found;
    const int i = blockIdx.y, s = src[i], d = dst[i];
    if (s < 0 || d < 0) return;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    bool bad = (uint32_t)s >= (uint32_t)items || (uint32_t)d >= (uint32_t)items;
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
        const int sj = src[j], dj = dst[j];
        if (sj >= 0 && dj >= 0) bad |= sj == d || (j < i && dj == d);
    }
    if (bad) found = 1;
    __syncthreads();
    if (found) {
        if (threadIdx.x == 0) raise_flag(error_flag);
        return;
    }
    const int plane = blockIdx.x / parts, part = blockIdx.x - plane * parts;
    char *base = pool + plane * plane_bytes + part * part_bytes;
    copy_chunks(base + s * item_bytes, base + d * item_bytes,
                min(part_bytes, item_bytes - part * part_bytes) / 16);
}

// The checks that all of these share.
int32_t check_book(const int32_t *table, const int32_t *lengths, const int32_t *refs,
                   const int32_t *free_pages, int64_t n, int64_t rows, int64_t width,
                   int64_t pages, int64_t page_size) {
    const int64_t lim = (int64_t)1 << 31;
    if (n < 0 || n >= ((int64_t)1 << 24) || rows <= 0 || rows >= kMaxRows || width <= 0 ||
        pages <= 0 || pages > kMaxPages || page_shift(page_size) < 0 ||
        width >= lim / page_size || rows * width > kMaxPages)
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

// Bytes that the bookkeeping workgroup copies by itself, done sooner than a second launch
// is (5 children of a row, pages of 4 KB a head in 2 planes of 2: with the call before and
// the one after it 27.3 us in two launches, 22.4 in one).
constexpr int64_t kOwnCopies = 256 << 10;

extern "C" int64_t qdc_pages_fork_workspace(int64_t n, int64_t page_size, int64_t planes,
                                            int64_t heads, int64_t token_bytes) {
    if (n <= 0 || n >= ((int64_t)1 << 24) || planes <= 0) return 0;
    const __int128 most = (__int128)n * planes * heads * page_size * token_bytes;
    return n <= kBook && most <= kOwnCopies ? 0 : 16 * n;
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
    // a workgroup per entry, plane, head and piece in a grid of fewer than 2^32 work-items
    if (planes < 0 ||
        (planes > 0 && (heads <= 0 || token_bytes <= 0 || token_bytes % 16 || planes >= 65536 ||
                        heads >= 65536 || planes * heads >= 65536 || token_bytes >= (1 << 20) ||
                        n * planes * heads * ceil_div(page_size * token_bytes, kBegun) >=
                            (1 << 24))))
        return QDC_ERR_SHAPE;
    const int64_t page_bytes = planes ? heads * page_size * token_bytes : 0;
    const int64_t bytes = pool_bytes(planes, pages, page_bytes);
    if (bytes < 0) return QDC_ERR_SHAPE;
    if (n == 0) return QDC_OK;
    const int64_t need = qdc_pages_fork_workspace(n, page_size, planes, heads, token_bytes);
    // without copies the list of them is in LDS and unused, whatever n is
    const bool own = need == 0;
    if (!parents || !children || (need && !workspace) || (planes > 0 && !pool)) return QDC_ERR_NULL;
    if (workspace_bytes < need || (need && !aligned16(workspace)) || !aligned16(pool))
        return QDC_ERR_SHAPE;
    const Range outs[7] = {QDC_BOOK_RANGES, {workspace, need}, {pool, bytes}};
    const Range ins[2] = {{parents, n * 4}, {children, n * 4}};
    if (any_alias(outs, 7, ins, 2)) return QDC_ERR_ALIAS;
    Copy *copies = own ? nullptr : reinterpret_cast<Copy *>(workspace);
    const Pool p = {(char *)pool, pages * page_bytes, page_bytes, token_bytes, (int)planes,
                    (int)heads};
    hipLaunchKernelGGL(pages_fork, dim3(1), dim3(kBook), bit_bytes(rows), stream,
                       make_book(table, lengths, refs, free_pages, n, rows, width, pages, page_size,
                                 error_flag), parents, children, copies, p);
    const int32_t status = launch_status();
    if (status != QDC_OK || own) return status;
    const int64_t pieces = ceil_div(page_size * token_bytes, kBegun);
    hipLaunchKernelGGL(copy_begun, dim3((uint32_t)n, (uint32_t)(planes * heads), (uint32_t)pieces),
                       dim3(kBlock), 0, stream, p, copies);
    return launch_status();
}

extern "C" int64_t qdc_pages_compact_workspace(int64_t pages) {
    return pages <= 0 || pages > kMaxPages ? 0 : 16 + 12 * pages;
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
    const int64_t most = ceil_div(pages, (int64_t)2) * planes * ceil_div(page_bytes, kPiece);
    const int64_t spread = ceil_div(rows * width + pages, (int64_t)kBlock);
    const int64_t want = most > spread ? most : spread;
    const uint32_t grid = (uint32_t)(want < kMoveGrid ? (want > 0 ? want : 1) : kMoveGrid);
    hipLaunchKernelGGL(pages_move, dim3(grid), dim3(kBlock), 0, stream, (char *)pool, planes,
                       pages * page_bytes, page_bytes, m, table, rows * width, free_pages,
                       (int)pages);
    return launch_status();
}

extern "C" int32_t qdc_copy_pages(void *pool, const int32_t *src, const int32_t *dst, int64_t n,
                                  int64_t planes, int64_t items, int64_t item_bytes,
                                  int32_t *error_flag, hipStream_t stream) {
    const int64_t lim = (int64_t)1 << 31;
    if (n < 0 || n > 4096 || planes < 0 || planes >= 65536 || items <= 0 || items >= lim ||
        item_bytes < 0 || item_bytes % 16 || item_bytes >= ((int64_t)1 << 40))
        return QDC_ERR_SHAPE;
    const int64_t bytes = pool_bytes(planes, items, item_bytes);
    if (bytes < 0) return QDC_ERR_SHAPE;
    if (n == 0 || planes == 0 || item_bytes == 0) return QDC_OK;
    if (!pool || !src || !dst) return QDC_ERR_NULL;
    if (!aligned16(pool)) return QDC_ERR_SHAPE;
    const Range outs[2] = {{pool, bytes}, {error_flag, error_flag ? 4 : 0}};
    const Range ins[2] = {{src, n * 4}, {dst, n * 4}};
    if (any_alias(outs, 2, ins, 2)) return QDC_ERR_ALIAS;
    // parts of a plane's item: enough workgroups for the chip, each at least 4 KB and at
    // most 64 KB, in a grid of fewer than 2^32 work-items
    const int64_t whole = n * planes * item_bytes;
    int64_t part = 4096;
    while (part < (64 << 10) && part < item_bytes && whole / part > 4096) part *= 2;
    int64_t parts, threads;
    for (;; part *= 2) {
        parts = ceil_div(item_bytes, part);
        threads = part / 16 < kPart ? part / 16 : kPart;
        if (n * planes * parts * threads < ((int64_t)1 << 32)) break;
        if (parts == 1) return QDC_ERR_SHAPE;
    }
    hipLaunchKernelGGL(copy_items, dim3((uint32_t)(planes * parts), (uint32_t)n),
                       dim3((uint32_t)threads), 0, stream, (char *)pool, src, dst, (int)n,
                       items * item_bytes, (int)items, item_bytes, part, (int)parts, error_flag);
    return launch_status();
}
