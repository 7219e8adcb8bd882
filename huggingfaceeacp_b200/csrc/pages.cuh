// The steps of a paged K/V cache whose book (table, lengths, reference counts)
// lives on the device: update (release, fork, grow), compact, write. No
// counterpart in the reference, whose cache is one contiguous window
// (Decoder.cpp:199-203).
//
// update and compact are two kernels each: one CTA does the bookkeeping on a
// few thousand integers, leaving a list of page copies in the workspace, and a
// grid copies the rows of all layers. Which page goes where is a prefix sum
// over ids, so the result does not depend on the order in which threads run;
// the only atomics add and subtract integers.
//
// Measured (B200): 3.54 GB of page moves in 590 us, 6.0 TB/s or 0.92 of the measured
// copy rate; 32 forks that copy their last page (119 MB read and written) 55 us, some
// 10 of them the bookkeeping; 131 MB of prompt rows written in 26 us. Small steps are
// bound by launches: 11 us on the GPU for a step of 16 sequences.
#pragma once

#include "common.cuh"

namespace hfk
{
constexpr int kPageLog = 6; // positions of a page: 64
constexpr int kPagePositions = 1 << kPageLog;
constexpr int kBookThreads = 1024;

struct PageCopy
{
    int source, target, rows;
};

// The cache as the kernels see it; layer_bytes and row_bytes are of one pool.
struct PageBook
{
    char* keys;
    char* values;
    long long layer_bytes;
    int row_bytes;
    int layers, pages, sequences, table_stride;
    int* table;
    int* lengths;
    int* refs;
    // workspace
    int* copy_count;
    PageCopy* copies; // [max(sequences, pages)]
    int* per_sequence; // [2][sequences]
    int* free_ids;     // [pages]
    int* renamed;      // [pages]
};

__device__ __forceinline__ bool page_there(int id, int pages)
{
    return (unsigned) id < (unsigned) pages;
}

// The table entries that a sequence of `length` positions uses.
__device__ __forceinline__ int pages_of(long long length, int stride)
{
    const long long n = (length + kPagePositions - 1) >> kPageLog;
    return n < 0 ? 0 : (n > stride ? stride : (int) n);
}

// Exclusive prefix sum over the CTA, and the CTA's total. All threads call it.
__device__ __forceinline__ int block_scan(int v, int* total)
{
    __shared__ int warps[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const int up = __shfl_up_sync(0xFFFFFFFFu, sum, o);
        if (lane >= o)
            sum += up;
    }
    __syncthreads(); // the last call's reads of `warps` are done
    if (lane == 31)
        warps[warp] = sum;
    __syncthreads();
    const int w = lane < (int) (blockDim.x >> 5) ? warps[lane] : 0;
    int before = lane < warp ? w : 0, all = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
    {
        before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
        all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
    }
    *total = all;
    return before + sum - v;
}

// The book's counts and lengths, the scratch and the call's lists in shared memory
// where they fit (kSmallBook words): one round trip to L2 brings them all, and the
// phases then run at shared memory's latency instead of L2's. Larger books stay where
// they are and are read past L1.
constexpr int kSmallBook = 48 * 1024;

__host__ __device__ constexpr long long book_words(long long pages, long long sequences)
{
    return 2 * pages + 7 * sequences; // refs, free ids; lengths, last, first, grow, forks, release
}

template <bool Small>
struct BookView
{
    int* lengths;
    int* refs;
    int* last;  // [sequences] scratch: a fork's length, then the page that a sequence would write into
    int* first; // [sequences] scratch: where its new pages begin among the free ones
    int* free_ids;
    const int* release;
    const int* forks;
    const int* grow;
    __device__ int at(const int* p, int i) const { return Small ? p[i] : __ldcg(&p[i]); }
    __device__ int length(int s) const { return at(lengths, s); }
    __device__ int ref(int id) const { return at(refs, id); }
};

template <bool Small>
__device__ __forceinline__ BookView<Small> open_book(const PageBook& b, int* shared, const int* release, int releases,
                                                     const int* forks, int fork_count, const int* grow)
{
    if (!Small)
        return {b.lengths, b.refs, b.per_sequence, b.per_sequence + b.sequences, b.free_ids, release, forks, grow};
    const int n = b.sequences;
    int* lists = shared + 2 * b.pages + 3 * n;
    const BookView<Small> v = {shared + 2 * b.pages, shared, shared + 2 * b.pages + n, shared + 2 * b.pages + 2 * n,
                               shared + b.pages, lists, lists + n, grow ? lists + 3 * n : nullptr};
    for (int i = threadIdx.x; i < n; i += kBookThreads)
    {
        v.lengths[i] = b.lengths[i];
        if (grow)
            lists[3 * n + i] = grow[i];
        if (i < releases)
            lists[i] = release[i];
        if (i < fork_count)
        {
            lists[n + 2 * i] = forks[2 * i];
            lists[n + 2 * i + 1] = forks[2 * i + 1];
        }
    }
    for (int i = threadIdx.x; i < b.pages; i += kBookThreads)
        v.refs[i] = b.refs[i];
    __syncthreads();
    return v;
}

template <bool Small>
__device__ __forceinline__ void close_book(const PageBook& b, const BookView<Small>& v)
{
    if (!Small)
        return;
    __syncthreads();
    for (int i = threadIdx.x; i < b.sequences; i += kBookThreads)
        b.lengths[i] = v.lengths[i];
    for (int i = threadIdx.x; i < b.pages; i += kBookThreads)
        b.refs[i] = v.refs[i];
}

// One CTA. What an earlier phase may have changed is read through L2 (__ldcg)
// where it is not in shared memory.
template <bool Small>
__global__ void __launch_bounds__(kBookThreads) pages_update_book(const PageBook b, const int* release, int releases,
                                                                  const int* forks, int fork_count, const int* grow,
                                                                  int* result)
{
    extern __shared__ int shared[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kWarps = kBookThreads / 32;
    pdl_wait();
    pdl_trigger();
    const BookView<Small> v = open_book<Small>(b, shared, release, releases, forks, fork_count, grow);

    for (int i = warp; i < releases; i += kWarps)
    {
        const int s = v.release[i];
        if ((unsigned) s >= (unsigned) b.sequences)
            continue;
        int length = 0;
        if (lane == 0)
            length = atomicExch(&v.lengths[s], 0); // a second listing finds 0
        length = __shfl_sync(0xFFFFFFFFu, length, 0);
        const int held = pages_of(length, b.table_stride);
        int* row = b.table + (size_t) s * b.table_stride;
        for (int j = lane; j < held; j += 32)
        {
            const int id = row[j];
            if (page_there(id, b.pages))
                atomicSub(&v.refs[id], 1);
            row[j] = -1;
        }
    }
    __syncthreads();

    // Forks: every pair's length is taken before any target is filled.
    int* fork_length = v.last;
    if (fork_count > 0)
    {
        for (int i = warp; i < fork_count; i += kWarps)
        {
            const int source = v.forks[2 * i], target = v.forks[2 * i + 1];
            bool ok = (unsigned) source < (unsigned) b.sequences && (unsigned) target < (unsigned) b.sequences
                      && v.length(target) <= 0;
            for (int e = lane; e < i && ok; e += 32)
                ok = v.forks[2 * e + 1] != target;
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (lane == 0)
                fork_length[i] = ok ? v.length(source) : 0;
        }
        __syncthreads();
        for (int i = warp; i < fork_count; i += kWarps)
        {
            const int length = v.at(fork_length, i);
            if (length <= 0)
                continue;
            const int held = pages_of(length, b.table_stride);
            const int* from = b.table + (size_t) v.forks[2 * i] * b.table_stride;
            int* to = b.table + (size_t) v.forks[2 * i + 1] * b.table_stride;
            for (int j = lane; j < held; j += 32)
            {
                const int id = __ldcg(&from[j]);
                to[j] = id;
                if (page_there(id, b.pages))
                    atomicAdd(&v.refs[id], 1);
            }
            if (lane == 0)
                v.lengths[v.forks[2 * i + 1]] = length;
        }
        __syncthreads();
    }

    // Growth: last[s] is the partly filled page that sequence s would write
    // into, -1 when there is none; it is copied while more than one sequence
    // holds it, those before s that have moved off it no longer counted.
    int* last = v.last;
    int* first = v.first;
    int wanted = 0, past = 0;
    if (grow)
    {
        for (int s = tid; s < b.sequences; s += kBookThreads)
        {
            const int length = max(v.length(s), 0);
            int id = -1;
            if (v.grow[s] > 0 && (length & (kPagePositions - 1)) && length >> kPageLog < b.table_stride)
                id = __ldcg(&b.table[(size_t) s * b.table_stride + (length >> kPageLog)]);
            last[s] = page_there(id, b.pages) && v.ref(id) > 1 ? id : -1;
        }
        __syncthreads();
        for (int base = 0; base < b.sequences; base += kBookThreads)
        {
            const int s = base + tid;
            int need = 0, over = 0;
            if (s < b.sequences && v.grow[s] > 0)
            {
                const int length = max(v.length(s), 0);
                const long long grown = (long long) length + v.grow[s];
                over = grown > (long long) b.table_stride * kPagePositions;
                need = over ? 0 : pages_of(grown, b.table_stride) - pages_of(length, b.table_stride);
                const int id = v.at(last, s);
                if (id >= 0)
                {
                    int holders = v.ref(id);
                    for (int e = 0; e < s; ++e)
                        holders -= v.at(last, e) == id;
                    need += holders > 1 ? 1 : 0;
                    if (holders > 1)
                        need |= 1 << 30; // the copy, kept beside the count
                }
            }
            int total;
            const int before = block_scan(need & 0x3FFFFFFF, &total);
            const int overs = __syncthreads_count(over);
            if (s < b.sequences)
                first[s] = (wanted + before) | (need & (1 << 30));
            wanted = min(wanted + total, 1 << 29); // need <= 2^20: no sum overflows; this many are never there
            past += overs;
        }
    }
    // The free ids, ascending, as far as they are wanted, and how many there are.
    int room = 0;
    for (int base = 0; base < b.pages; base += 4 * kBookThreads)
    {
        int free_here[4], n = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            const int id = base + 4 * tid + k;
            free_here[k] = id < b.pages && v.ref(id) <= 0;
            n += free_here[k];
        }
        int total;
        int at = room + block_scan(n, &total);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (free_here[k])
            {
                if (at < wanted)
                    v.free_ids[at] = base + 4 * tid + k;
                ++at;
            }
        room += total;
    }
    __syncthreads();
    const bool fits = wanted <= room && past == 0;
    int copied = 0;
    if (grow && fits)
        for (int base = 0; base < b.sequences; base += kBookThreads)
        {
            const int s = base + tid;
            const bool grows = s < b.sequences && v.grow[s] > 0;
            const int entry = grows ? v.at(first, s) : 0;
            const bool copies = entry & (1 << 30);
            int total;
            const int slot = copied + block_scan(copies, &total);
            copied += total;
            if (!grows)
                continue;
            int* row = b.table + (size_t) s * b.table_stride;
            const int length = max(v.length(s), 0);
            const int held = pages_of(length, b.table_stride);
            const int need = pages_of((long long) length + v.grow[s], b.table_stride) - held;
            int at = entry & 0x3FFFFFFF;
            if (copies)
            {
                const int id = v.at(last, s), fresh = v.at(v.free_ids, at++);
                b.copies[slot] = {id, fresh, length & (kPagePositions - 1)};
                row[held - 1] = fresh;
                v.refs[fresh] = 1;
                atomicSub(&v.refs[id], 1);
            }
            for (int j = 0; j < need; ++j)
            {
                const int fresh = v.at(v.free_ids, at + j);
                row[held + j] = fresh;
                v.refs[fresh] = 1;
            }
            v.lengths[s] = length + v.grow[s];
        }
    if (tid == 0)
    {
        *b.copy_count = copied;
        result[0] = fits ? room - wanted : room;
        result[1] = max(wanted - room, 0);
        result[2] = past;
    }
    close_book<Small>(b, v);
}

// One CTA: counts the held pages, pairs those above the count with the free
// ids below it, renames the table's entries and moves the counts.
template <bool Small>
__global__ void __launch_bounds__(kBookThreads) pages_compact_book(const PageBook b, int* live_out)
{
    extern __shared__ int shared[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_trigger();
    const BookView<Small> v = open_book<Small>(b, shared, nullptr, 0, nullptr, 0, nullptr);
    int live = 0;
    for (int base = 0; base < b.pages; base += kBookThreads)
        live += __syncthreads_count(base + tid < b.pages && v.ref(base + tid) > 0);
    int leaves = 0, holes = 0;
    for (int base = 0; base < b.pages; base += kBookThreads)
    {
        const int id = base + tid;
        const bool held = id < b.pages && v.ref(id) > 0;
        const bool leaves_here = held && id >= live, hole = id < live && !held;
        int total;
        const int both = block_scan(leaves_here | hole << 16, &total); // 1024 of each at most
        const int at = leaves + (both & 0xFFFF), hole_at = holes + (both >> 16);
        leaves += total & 0xFFFF;
        holes += total >> 16;
        if (leaves_here)
            b.copies[at].source = id;
        if (hole)
            v.free_ids[hole_at] = id;
    }
    __syncthreads();
    for (int i = tid; i < leaves; i += kBookThreads)
    {
        const int source = __ldcg(&b.copies[i].source), target = v.at(v.free_ids, i);
        b.copies[i] = {source, target, kPagePositions};
        b.renamed[source] = target;
        v.refs[target] = v.ref(source);
        v.refs[source] = 0;
    }
    __syncthreads();
    for (int s = warp; s < b.sequences; s += kBookThreads / 32)
    {
        int* row = b.table + (size_t) s * b.table_stride;
        const int held = pages_of(v.length(s), b.table_stride);
        for (int j = lane; j < held; j += 32)
        {
            const int id = row[j];
            if (page_there(id, b.pages) && id >= live)
                row[j] = __ldcg(&b.renamed[id]);
        }
    }
    if (tid == 0)
    {
        *b.copy_count = leaves;
        *live_out = live;
    }
    close_book<Small>(b, v);
}

// The rows in use of every listed page, in all layers, keys and values, in pieces of
// 32 KB that the grid's CTAs take in turn: eight 16-byte loads in flight a thread.
// Bound by HBM: each byte is read and written once.
__global__ void __launch_bounds__(256) pages_copy_rows(const PageBook b)
{
    constexpr int kPiece = 8 * 256; // 16-byte words
    pdl_wait();
    const int words = kPagePositions * (b.row_bytes / 16), pieces = (words + kPiece - 1) / kPiece;
    const long long units = (long long) *(volatile const int*) b.copy_count * b.layers * 2 * pieces;
    for (long long u = blockIdx.x; u < units; u += gridDim.x)
    {
        const int piece = (int) (u % pieces);
        const long long pool_of = u / pieces;
        const PageCopy c = b.copies[pool_of / (2 * b.layers)];
        const int n = c.rows * (b.row_bytes / 16), begin = piece * kPiece + threadIdx.x;
        if (piece * kPiece >= n)
            continue;
        const int layer = (int) (pool_of / 2 % b.layers);
        char* pool = (pool_of & 1 ? b.values : b.keys) + (long long) layer * b.layer_bytes;
        const uint4* from = reinterpret_cast<const uint4*>(pool) + (size_t) c.source * words;
        uint4* to = reinterpret_cast<uint4*>(pool) + (size_t) c.target * words;
        uint4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (begin + k * 256 < n)
                x[k] = __ldcs(from + begin + k * 256);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (begin + k * 256 < n)
                __stcs(to + begin + k * 256, x[k]);
    }
}

struct PageWrite
{
    char* keys; // the layer's
    char* values;
    const char* k;
    const char* v;
    long long k_stride, v_stride; // bytes
    int row_bytes, pages, sequences, table_stride;
    const int* table;
    const int* lengths;
    const int* offsets;
    const int* index;
    int rows, source_rows;
};

// offsets[s] as the calls take it: within [0, rows].
__device__ __forceinline__ int bounded_offset(const int* offsets, int s, int rows)
{
    return min(max(offsets[s], 0), rows);
}

// The sequence whose rows hold r: the last s with offsets[s] <= r, -1 for none.
__device__ __forceinline__ int sequence_of(const int* offsets, int sequences, int rows, int r)
{
    int low = -1, high = sequences; // offsets[low] <= r < offsets[high]
    while (high - low > 1)
    {
        const int mid = (low + high) / 2;
        if (bounded_offset(offsets, mid, rows) <= r)
            low = mid;
        else
            high = mid;
    }
    return low >= 0 && low < sequences && r < bounded_offset(offsets, low + 1, rows) ? low : -1;
}

// One warp a row.
__global__ void __launch_bounds__(256) pages_write_rows(const PageWrite w)
{
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= w.rows)
        return;
    const int s = sequence_of(w.offsets, w.sequences, w.rows, r);
    if (s < 0)
        return;
    const long long position = (long long) w.lengths[s] - bounded_offset(w.offsets, s + 1, w.rows) + r;
    if (position < 0 || position >= (long long) w.table_stride << kPageLog)
        return;
    const int id = w.table[(size_t) s * w.table_stride + (position >> kPageLog)];
    const int source = w.index ? w.index[r] : r;
    if (!page_there(id, w.pages) || (unsigned) source >= (unsigned) w.source_rows)
        return;
    const size_t at = ((size_t) id * kPagePositions + (position & (kPagePositions - 1))) * w.row_bytes;
    const uint4* k = reinterpret_cast<const uint4*>(w.k + source * w.k_stride);
    const uint4* v = reinterpret_cast<const uint4*>(w.v + source * w.v_stride);
    uint4* keys = reinterpret_cast<uint4*>(w.keys + at);
    uint4* values = reinterpret_cast<uint4*>(w.values + at);
    for (int i = lane; i < w.row_bytes / 16; i += 32)
    {
        keys[i] = k[i];
        values[i] = v[i];
    }
}
} // namespace hfk
