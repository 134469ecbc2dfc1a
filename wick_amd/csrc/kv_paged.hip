// KV caches in pages that sequences share: rows appended, and what is done to pages themselves -- sequences forked and cut, pages taken for new rows (with
// a copy of a page that others hold too), the pool moved together.  Who holds what is in the table, lens and refs of wick_rocm_kv_pages, all on the device.
#include <algorithm>

#include "kv_paged_device.h"
#include "wick_rocm_internal.h"

namespace wick_rocm {

namespace {

// ---- append --------------------------------------------------------------------------------------
// One thread a 16-byte load of each source; bound by memory (2002 tokens of 8 heads of 64 in f32, 16 MB: 4.8 us, 3.4 TB/s), and by the launch where there are few
// tokens (64: 3.8 us).
struct PagedAppendArgs {
    const float* src[2];  // keys, values
    void* pages[2];
    PagedRows rows;
    uint32_t n, n_kv_heads, head_dim, stride;
};

template <typename KV>
__global__ __launch_bounds__(256) void kv_paged_append_kernel(PagedAppendArgs a) {
    const uint32_t quads = a.n_kv_heads * a.head_dim / 4u;
    const uint64_t at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (at >= (uint64_t)a.n * quads) return;
    const uint32_t j = (uint32_t)(at / quads), quad = (uint32_t)(at % quads), c = 4u * quad / a.head_dim, i = 4u * quad % a.head_dim;
    uint32_t page;
    const uint32_t row = paged_row(a.rows, j, page);
    if (row == WICK_ROCM_NO_ROW || page >= a.rows.n_pages) return;
    const size_t to = paged_at(a.rows, page, row, a.n_kv_heads, c, a.head_dim) + i;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        const float4 x = *reinterpret_cast<const float4*>(a.src[which] + (size_t)j * a.stride + 4u * quad);
        KV* const p = static_cast<KV*>(a.pages[which]) + to;
        if constexpr (sizeof(KV) == 4) {
            *reinterpret_cast<float4*>(p) = x;
        } else {
            const h4 h = {(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w};
            *reinterpret_cast<h4*>(p) = h;
        }
    }
}

// ---- fork, free ----------------------------------------------------------------------------------
// A table's columns are independent of each other: a workgroup takes a few of them for all sequences, so that it has read every
// parent's entries before it writes any, and one launch does it in place.  One workgroup more does the same with lens.  Bound by its round trips: 3.9 us for 17
// sequences of 32 pages, 4.9 for 8 of 1000.
constexpr uint32_t kForkEntries = 8192;  // of a workgroup (LDS); a power of two, at least the most sequences
struct PagedForkArgs {
    uint32_t *table, *lens, *refs;
    const uint32_t* parents;
    uint32_t n_seqs, max_pages, n_pages, columns;
};

__global__ __launch_bounds__(256) void kv_pages_fork_kernel(PagedForkArgs a) {
    __shared__ uint32_t old[kForkEntries];
    const bool is_lens = blockIdx.x == gridDim.x - 1u;
    const uint32_t first = blockIdx.x * a.columns, columns = is_lens ? 1u : min(a.columns, a.max_pages - first);
    uint32_t* const entries = is_lens ? a.lens : a.table + first;
    const uint32_t stride = is_lens ? 1u : a.max_pages, none = is_lens ? 0u : WICK_ROCM_NO_PAGE;
    for (uint32_t i = threadIdx.x; i < a.n_seqs * columns; i += 256u) old[i] = entries[(size_t)(i / columns) * stride + i % columns];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.n_seqs * columns; i += 256u) {
        const uint32_t s = i / columns, parent = a.parents[s];
        if (parent == s) continue;
        const uint32_t was = old[i], is = parent < a.n_seqs ? old[parent * columns + i % columns] : none;
        if (was == is) continue;
        entries[(size_t)s * stride + i % columns] = is;
        if (is_lens) continue;
        if (was < a.n_pages) atomicSub(&a.refs[was], 1u);
        if (is < a.n_pages) atomicAdd(&a.refs[is], 1u);
    }
}

struct PagedFreeArgs {
    uint32_t *table, *lens, *refs;
    const uint32_t* rows;
    uint32_t n_seqs, max_pages, n_pages, page_shift;
};

__global__ __launch_bounds__(256) void kv_pages_free_kernel(PagedFreeArgs a) {
    const uint64_t all = (uint64_t)a.n_seqs * a.max_pages;
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256u) {
        const uint32_t s = (uint32_t)(i / a.max_pages), p = (uint32_t)(i % a.max_pages), rows = a.rows[s];
        if (p == 0 && rows < a.lens[s]) a.lens[s] = rows;
        if (p < pages_of(rows, a.page_shift)) continue;
        const uint32_t page = a.table[i];
        if (page == WICK_ROCM_NO_PAGE) continue;
        a.table[i] = WICK_ROCM_NO_PAGE;
        if (page < a.n_pages) atomicSub(&a.refs[page], 1u);
    }
}

// ---- the plan of a reservation or a compaction: one workgroup --------------------------------------
// A chain of round trips to memory (lengths, the table's entry, its page's count; what is written) and of barriers; refs are read a run of pages a thread, of
// the first 16384 pages once, at the start.  A row for each of 16 continuations (a shared page copied) takes 9.2 us, 2002 rows for one of 32 sequences 6.5, a compaction
// of 8000 pages 4.9.
constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr uint32_t kRun = 16;                    // consecutive pages of a thread at a time
constexpr uint32_t kListed = 4096;               // pages of a list that are in LDS; those behind them in memory
constexpr uint32_t kSeqs = 4;                    // sequences of a thread: 4096 in all
constexpr uint32_t kShared = 2 * kSeqs * kPlanThreads;  // slots for the pages that are shared and written to

// Sum over the workgroup's threads in front of this one, and over all of them.  `slots`: kPlanWaves, of this call alone until the next barrier.
__device__ __forceinline__ uint32_t sum_before(uint32_t v, uint32_t* slots, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), upto = lanes_upto(v);
    if (lane == 63u) slots[wave] = upto;
    __syncthreads();
    const uint32_t sums = lanes_upto(lane < kPlanWaves ? slots[lane] : 0u);
    total = (uint32_t)__builtin_amdgcn_readlane((int)sums, 63);
    return upto - v + (wave > 0 ? (uint32_t)__builtin_amdgcn_readlane((int)sums, (int)wave - 1) : 0u);
}

// Bits of the pages [first, first + kRun) that are free; those behind the last page are not.
__device__ __forceinline__ uint32_t free_bits(const uint32_t* refs, uint64_t first, uint32_t n_pages) {
    uint32_t bits = 0;
    if (first + kRun <= n_pages) {
#pragma unroll
        for (uint32_t i = 0; i < kRun; i += 4) {
            const u32x4_a4 x = *reinterpret_cast<const u32x4_a4*>(refs + first + i);
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) bits |= (uint32_t)(x.v[e] == 0) << (i + e);
        }
    } else {
        for (uint32_t i = 0; first + i < n_pages; i++) bits |= (uint32_t)(refs[first + i] == 0) << i;
    }
    return bits;
}

struct PagedPlanArgs {
    uint32_t *table, *lens, *refs, *start, *moves, *list;  // list: n_pages words behind the moves
    const uint32_t* counts;
    uint32_t n_seqs, max_pages, n_pages, page_shift;
};

// Pages for the new rows of every sequence.  A partial last page with c writers and r holders: where c = r the first writer keeps it and r - 1 copy, else all c
// do.  Who is who is found in LDS, by the page's slot of a hash table twice as large as all sequences, for pages that are shared alone.
__global__ __launch_bounds__(kPlanThreads) void kv_pages_reserve_kernel(PagedPlanArgs a) {
    __shared__ uint32_t page_of[kShared], writers[kShared], first_of[kShared], list[kListed], slots[3][kPlanWaves];
    const uint32_t R = 1u << a.page_shift;
    const uint64_t capacity = (uint64_t)a.max_pages << a.page_shift;
    uint32_t len[kSeqs], count[kSeqs], page[kSeqs], held[kSeqs], need[kSeqs];
    uint32_t bits = free_bits(a.refs, threadIdx.x * kRun, a.n_pages);
    bool too_long = false, copies[kSeqs], shared = false;
#pragma unroll
    for (uint32_t k = 0; k < kSeqs; k++) {  // consecutive sequences a thread, in order
        const uint32_t s = threadIdx.x * kSeqs + k;
        len[k] = s < a.n_seqs ? a.lens[s] : 0, count[k] = s < a.n_seqs ? a.counts[s] : 0;
    }
#pragma unroll
    for (uint32_t k = 0; k < kSeqs; k++) {
        const uint32_t s = threadIdx.x * kSeqs + k;
        too_long = too_long || (uint64_t)len[k] + count[k] > capacity;
        page[k] = count[k] != 0 && len[k] % R != 0 && len[k] < capacity ? a.table[(size_t)s * a.max_pages + (len[k] >> a.page_shift)] : WICK_ROCM_NO_PAGE;
    }
#pragma unroll
    for (uint32_t k = 0; k < kSeqs; k++) {
        held[k] = page[k] < a.n_pages ? a.refs[page[k]] : 0u;
        shared = shared || held[k] > 1u, copies[k] = held[k] > 1u;
    }
    uint32_t move = 0, moves = 0;  // this thread's first one, and all: in the sequences' order
    if (__syncthreads_or(shared)) {
        uint32_t size = 64;
        while (size < 2u * a.n_seqs) size *= 2u;
        for (uint32_t i = threadIdx.x; i < size; i += kPlanThreads) page_of[i] = WICK_ROCM_NO_PAGE, writers[i] = 0, first_of[i] = WICK_ROCM_NO_PAGE;
        __syncthreads();
        uint32_t slot[kSeqs];
#pragma unroll
        for (uint32_t k = 0; k < kSeqs; k++) {
            if (!copies[k]) continue;
            slot[k] = page[k] * 0x9e3779b1u >> 8 & (size - 1u);
            for (uint32_t is; (is = atomicCAS(&page_of[slot[k]], WICK_ROCM_NO_PAGE, page[k])) != WICK_ROCM_NO_PAGE && is != page[k];)  // (at most half of the slots are taken)
                slot[k] = (slot[k] + 1u) & (size - 1u);
            atomicAdd(&writers[slot[k]], 1u), atomicMin(&first_of[slot[k]], threadIdx.x * kSeqs + k);
        }
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < kSeqs; k++)
            if (copies[k]) copies[k] = writers[slot[k]] != held[k] || first_of[slot[k]] != threadIdx.x * kSeqs + k;
        uint32_t mine = 0;
#pragma unroll
        for (uint32_t k = 0; k < kSeqs; k++) mine += copies[k];
        move = sum_before(mine, slots[2], moves);
    }
    uint32_t mine = 0;
#pragma unroll
    for (uint32_t k = 0; k < kSeqs; k++) {
        need[k] = count[k] == 0 ? 0 : pages_of((uint64_t)len[k] + count[k], a.page_shift) - pages_of(len[k], a.page_shift) + copies[k];
        mine += need[k];
    }
    const bool fits_table = !__syncthreads_or(too_long);
    uint32_t wanted;
    uint32_t at = sum_before(mine, slots[0], wanted);
    // the lowest free pages, as many as are wanted
    uint32_t found = 0;
    for (uint64_t base = 0; fits_table && base < a.n_pages && found < wanted; base += kRun * kPlanThreads) {
        const uint64_t first = base + threadIdx.x * kRun;
        if (base != 0) bits = free_bits(a.refs, first, a.n_pages);
        uint32_t all;
        uint32_t to = found + sum_before(__popc(bits), slots[1], all);
        for (; bits != 0 && to < wanted; bits &= bits - 1u, to++) (to < kListed ? list[to] : a.list[to]) = (uint32_t)first + __ffs(bits) - 1u;
        found += all;
        __syncthreads();  // (slots are read, the list is written)
    }
    if (!fits_table || found < wanted) {  // nothing changes
#pragma unroll
        for (uint32_t k = 0; k < kSeqs; k++)
            if (const uint32_t s = threadIdx.x * kSeqs + k; s < a.n_seqs) a.start[s] = WICK_ROCM_NO_ROW;
        if (threadIdx.x == 0) *reinterpret_cast<uint4*>(a.moves) = make_uint4(0, fits_table ? wanted - found : 0xffffffffu, 0, 0);
        return;
    }
    // where a sequence's new pages begin, in the list and in its row of the table (in place of what is in LDS no longer needed)
    uint32_t* const begin = page_of;
    uint32_t* const entry = writers;
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kSeqs; k++) {
        const uint32_t s = threadIdx.x * kSeqs + k;
        begin[s] = at, entry[s] = pages_of(len[k], a.page_shift) - copies[k];
        if (s < a.n_seqs) a.start[s] = count[k] == 0 ? WICK_ROCM_NO_ROW : len[k];
        if (count[k] == 0) continue;
        a.lens[s] = len[k] + count[k];
        if (copies[k]) {
            atomicSub(&a.refs[page[k]], 1u);
            *reinterpret_cast<uint4*>(a.moves + 4u + 4u * move++) = make_uint4(page[k], at < kListed ? list[at] : a.list[at], len[k] % R, 0);
        }
        at += need[k];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < wanted; i += kPlanThreads) {  // the last sequence that begins at or in front of it
        uint32_t low = 0, high = a.n_seqs;
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2u;
            (begin[mid] <= i ? low : high) = mid;
        }
        const uint32_t to = i < kListed ? list[i] : a.list[i];
        a.table[(size_t)low * a.max_pages + entry[low] + (i - begin[low])] = to, a.refs[to] = 1;
    }
    if (threadIdx.x == 0) *reinterpret_cast<uint4*>(a.moves) = make_uint4(moves, 0, 0, 0);
}

// With U pages in use: the i-th page in use at U or above goes to the i-th free one below.
__global__ __launch_bounds__(kPlanThreads) void kv_pages_compact_kernel(PagedPlanArgs a) {
    __shared__ uint32_t from_list[kListed], to_list[kListed], slots[2][kPlanWaves];
    const uint32_t early = free_bits(a.refs, threadIdx.x * kRun, a.n_pages);
    uint32_t free = __popc(early);
    for (uint64_t base = kRun * kPlanThreads; base < a.n_pages; base += kRun * kPlanThreads) free += __popc(free_bits(a.refs, base + threadIdx.x * kRun, a.n_pages));
    uint32_t all;
    sum_before(free, slots[0], all);
    const uint32_t used = a.n_pages - all;
    uint32_t holes = 0, movers = 0;
    for (uint64_t base = 0; base < a.n_pages; base += kRun * kPlanThreads) {
        const uint64_t first = base + threadIdx.x * kRun;
        const uint32_t bits = base == 0 ? early : free_bits(a.refs, first, a.n_pages);
        const uint32_t inside = first >= a.n_pages ? 0u : first + kRun <= a.n_pages ? 0xffffu : (1u << (a.n_pages - first)) - 1u;
        const uint32_t below = first >= used ? 0u : first + kRun <= used ? 0xffffu : (1u << (used - first)) - 1u;
        uint32_t hole = bits & below, mover = ~bits & inside & ~below, n;
        const uint32_t before = sum_before(__popc(hole) | __popc(mover) << 16, slots[1], n);  // (at most 2^14 each)
        uint32_t to = holes + (before & 0xffffu), from = movers + (before >> 16);
        for (; hole != 0; hole &= hole - 1u, to++) (to < kListed ? to_list[to] : a.moves[4u + 4u * to + 1u]) = (uint32_t)first + __ffs(hole) - 1u;
        for (; mover != 0; mover &= mover - 1u, from++) (from < kListed ? from_list[from] : a.moves[4u + 4u * from]) = (uint32_t)first + __ffs(mover) - 1u;
        holes += n & 0xffffu, movers += n >> 16;
        __syncthreads();
    }
    for (uint32_t m = threadIdx.x; m < movers; m += kPlanThreads) {
        uint32_t* const move = a.moves + 4u + 4u * m;
        const uint32_t from = m < kListed ? from_list[m] : move[0], to = m < kListed ? to_list[m] : move[1];
        *reinterpret_cast<uint4*>(move) = make_uint4(from, to, 1u << a.page_shift, 0);
        a.refs[to] = a.refs[from], a.refs[from] = 0;
        a.list[from] = to;
    }
    if (threadIdx.x == 0) *reinterpret_cast<uint4*>(a.moves) = make_uint4(movers, used, 0, 0);
}

// ---- pages moved -----------------------------------------------------------------------------------
// A workgroup takes 1024 consecutive 16-byte pieces of a page in one plane, of one move after the other; for a compaction, the table's entries behind them.
// Bound by memory: 393 MB read and written in 81 us, 4.8 TB/s, the rate of a large copy; 50 MB in 11 us.
struct PagedCopyArgs {
    char* base;
    size_t plane_bytes;
    const uint32_t* moves;
    uint32_t* table;  // entries from moves[1] on are replaced by `list` of them (null: none)
    const uint32_t* list;
    uint32_t max_moves, n_pages, pieces, parts, row_shift, page_shift;  // pieces: of a page; parts: units of them; row_shift: pieces of a row of one head
    uint64_t entries;
};
constexpr uint32_t kUnit = 1024;

__global__ __launch_bounds__(256) void kv_pages_copy_kernel(PagedCopyArgs a) {
    const uint32_t moves = min(a.moves[0], a.max_moves), plane = blockIdx.x / a.parts, first = blockIdx.x % a.parts * kUnit + threadIdx.x;
    uint4* const pages = reinterpret_cast<uint4*>(a.base + plane * a.plane_bytes) + first;
    for (uint32_t m = blockIdx.y; m < moves; m += gridDim.y) {
        const uint4 move = *reinterpret_cast<const uint4*>(a.moves + 4u + 4u * (size_t)m);
        if (move.x >= a.n_pages || move.y >= a.n_pages) continue;
        const uint4* const from = pages + (size_t)move.x * a.pieces;
        uint4* const to = pages + (size_t)move.y * a.pieces;
        const auto takes = [&](uint32_t i) { return first + i < a.pieces && ((first + i) >> a.row_shift & ((1u << a.page_shift) - 1u)) < move.z; };
        uint4 x0, x1, x2, x3;
        const bool t0 = takes(0), t1 = takes(256), t2 = takes(512), t3 = takes(768);
        if (t0) x0 = from[0];
        if (t1) x1 = from[256];
        if (t2) x2 = from[512];
        if (t3) x3 = from[768];
        if (t0) to[0] = x0;
        if (t1) to[256] = x1;
        if (t2) to[512] = x2;
        if (t3) to[768] = x3;
    }
    if (a.table == nullptr) return;
    const uint32_t used = a.moves[1];
    const uint64_t at = ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256u + threadIdx.x, step = (uint64_t)gridDim.x * gridDim.y * 256u;
    for (uint64_t i = at; i < a.entries; i += step) {
        const uint32_t page = a.table[i];
        if (page >= used && page < a.n_pages) a.table[i] = a.list[page];
    }
}

constexpr uint32_t kCopyGroups = 2048;  // workgroups of a launch that copies, or a round of its planes

uint32_t page_shift(const wick_rocm_kv_pages& p) { return (uint32_t)__builtin_ctz(p.page_rows); }

size_t most_moves(const wick_rocm_kv_pages& p) { return std::max(p.n_seqs, p.n_pages / 2u); }

uint32_t blocks(uint64_t threads, uint32_t most) { return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(most, (threads + 255u) / 256u)); }

hipError_t launch_copy(const wick_rocm_kv_pages& p, const wick_rocm_kv_planes* planes, const uint32_t* d_moves, uint32_t max_moves, bool table, const Launch& L) {
    PagedCopyArgs a{};
    a.moves = d_moves, a.n_pages = p.n_pages, a.page_shift = page_shift(p), a.parts = 1;
    uint32_t x = 1, y = 1;
    if (planes) {
        const uint32_t row_pieces = planes->head_dim * (planes->kv_dtype == WICK_ROCM_KV_F16 ? 2u : 4u) / 16u;
        a.base = static_cast<char*>(planes->d_base), a.plane_bytes = planes->plane_bytes, a.max_moves = max_moves;
        a.row_shift = (uint32_t)__builtin_ctz(row_pieces), a.pieces = planes->n_kv_heads * p.page_rows * row_pieces, a.parts = (a.pieces + kUnit - 1u) / kUnit;
        x = planes->n_planes * a.parts;
        y = std::min(max_moves, std::max(1u, kCopyGroups / x));
    }
    if (table) {
        a.table = p.d_table, a.list = d_moves + 4u + 4u * most_moves(p), a.entries = (uint64_t)p.n_seqs * p.max_pages;
        y = std::max(y, std::min(blocks(a.entries, kCopyGroups) / x, 65535u));
    }
    return launch_kernel(L, kFamOther, kv_pages_copy_kernel, dim3(x, std::max(y, 1u)), dim3(256), a);
}

}  // namespace

hipError_t launch_kv_paged_append(const wick_rocm_kv_pages& p, const float* d_k, const float* d_v, uint32_t kv_stride, void* d_k_pages, void* d_v_pages,
                                  bool kv_f16, const uint32_t* d_start, const uint32_t* d_first, uint32_t n, uint32_t n_kv_heads, uint32_t head_dim,
                                  const Launch& L) {
    if (n == 0) return hipSuccess;
    const PagedAppendArgs a{{d_k, d_v}, {d_k_pages, d_v_pages}, {p.d_table, d_start, d_first, p.n_seqs, p.max_pages, p.n_pages, page_shift(p)}, n, n_kv_heads,
                            head_dim, kv_stride};
    const uint64_t threads = (uint64_t)n * (n_kv_heads * head_dim / 4u);
    const dim3 grid((uint32_t)((threads + 255u) / 256u));
    return kv_f16 ? launch_kernel(L, kFamOther, kv_paged_append_kernel<_Float16>, grid, dim3(256), a)
                  : launch_kernel(L, kFamOther, kv_paged_append_kernel<float>, grid, dim3(256), a);
}

hipError_t launch_kv_pages_fork(const wick_rocm_kv_pages& p, const uint32_t* d_parents, const Launch& L) {
    uint32_t columns = 16;
    while (columns > 1 && columns * p.n_seqs > kForkEntries) columns /= 2u;
    const PagedForkArgs a{p.d_table, p.d_lens, p.d_refs, d_parents, p.n_seqs, p.max_pages, p.n_pages, columns};
    return launch_kernel(L, kFamOther, kv_pages_fork_kernel, dim3((p.max_pages + columns - 1u) / columns + 1u), dim3(256), a);
}

hipError_t launch_kv_pages_free(const wick_rocm_kv_pages& p, const uint32_t* d_rows, const Launch& L) {
    const PagedFreeArgs a{p.d_table, p.d_lens, p.d_refs, d_rows, p.n_seqs, p.max_pages, p.n_pages, page_shift(p)};
    return launch_kernel(L, kFamOther, kv_pages_free_kernel, dim3(blocks((uint64_t)p.n_seqs * p.max_pages, 2048u)), dim3(256), a);
}

size_t kv_pages_moves_words(const wick_rocm_kv_pages& p) { return 4 + 4 * most_moves(p) + p.n_pages; }

hipError_t launch_kv_pages_reserve(const wick_rocm_kv_pages& p, const uint32_t* d_counts, uint32_t* d_start, uint32_t* d_moves, const wick_rocm_kv_planes* planes,
                                   const Launch& L) {
    const PagedPlanArgs a{p.d_table, p.d_lens, p.d_refs, d_start, d_moves, d_moves + 4u + 4u * most_moves(p), d_counts, p.n_seqs, p.max_pages, p.n_pages, page_shift(p)};
    hipError_t e = launch_kernel(L, kFamOther, kv_pages_reserve_kernel, dim3(1), dim3(kPlanThreads), a);
    return e != hipSuccess || !planes ? e : launch_copy(p, planes, d_moves, p.n_seqs, false, L);
}

hipError_t launch_kv_pages_compact(const wick_rocm_kv_pages& p, uint32_t* d_moves, const wick_rocm_kv_planes* planes, const Launch& L) {
    const PagedPlanArgs a{p.d_table, p.d_lens, p.d_refs, nullptr, d_moves, d_moves + 4u + 4u * most_moves(p), nullptr, p.n_seqs, p.max_pages, p.n_pages, page_shift(p)};
    hipError_t e = launch_kernel(L, kFamOther, kv_pages_compact_kernel, dim3(1), dim3(kPlanThreads), a);
    return e != hipSuccess ? e : launch_copy(p, planes, d_moves, p.n_pages / 2u, true, L);
}

hipError_t launch_kv_pages_copy(const wick_rocm_kv_pages& p, const wick_rocm_kv_planes& planes, const uint32_t* d_moves, uint32_t max_moves, const Launch& L) {
    return max_moves == 0 ? hipSuccess : launch_copy(p, &planes, d_moves, max_moves, false, L);
}

}  // namespace wick_rocm
