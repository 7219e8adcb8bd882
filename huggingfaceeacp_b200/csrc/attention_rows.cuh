// Attention of one query row by one warp, for the packed prompts
// (hf_attention_packed) and the drafted trees over a paged cache
// (hf_attention_tree): what each row attends to, and the plain row itself.
//
// Row (r, h) attends to a list of keys: its prompt's rows up to its own, or its
// sequence's cached positions and then the drafted nodes on its path. The warp
// takes 32 keys at a time: lane c holds channels [8 c, 8 c + 8) of the query,
// the 32 scores are warp sums left in the lanes, the running maximum m and sum
// l follow the blocks (p = 2^(s - m), the sums so far scaled by 2^(m_old -
// m_new)), and each block's weighted values are summed apart and then added to
// the row, so that no fp32 chain is longer than 32 + keys / 32. A key that the
// row does not attend to is not read, whatever it holds. A row that attends to
// nothing is 0; one whose every score is minus infinity is NaN, as by the formula.
#pragma once

#include "common.cuh"
#include "pages.cuh"

#include <cuda_bf16.h>

namespace hfk
{
constexpr int kTreeNodes = 64;

// What both calls hand to the kernels; strides in elements.
struct AttnCall
{
    const void* q;
    const void* k;
    const void* v;
    void* out;
    long long q_stride, k_stride, v_stride, out_stride;
    const int* offsets;
    int sequences, rows, heads, kv_heads, group, width;
    float scale_log2; // scale * log2(e)
    // a tree's
    const int* parents;
    const void* key_pages; // the layer's
    const void* value_pages;
    const int* table;
    const int* lengths;
    int pages, table_stride, max_nodes, max_length;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8])
{
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__half>(const __half* p, float (&x)[8])
{
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[8])
{
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

// Two fp32 as one 32-bit pair of T, the first in the low half, to nearest even.
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The row's only rounding to T.
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8])
{
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_pair<T>(x[0], x[1]), pack_pair<T>(x[2], x[3]),
                                              pack_pair<T>(x[4], x[5]), pack_pair<T>(x[6], x[7]));
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8])
{
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// What a row attends to: keys 0 .. cached - 1 in the cache, then `drafted` rows
// from row `first` on, of which those in `path` (a bit each; all of them for a
// prompt, where drafted is the row's place + 1).
struct RowKeys
{
    int cached, first, drafted;
    unsigned long long path;
    const int* table; // the sequence's row
};

// Bit i set for the nodes on the path from node n up (n < 64 nodes of a tree,
// parents within the tree; a parent that is not before its child ends the path).
template <typename Int>
__device__ __forceinline__ unsigned long long tree_path(const Int* parents, int n)
{
    unsigned long long path = 0;
    for (int i = n; i >= 0;)
    {
        path |= 1ull << i;
        const int up = parents[i];
        i = up < i ? up : -1;
    }
    return path;
}

// The sequence whose rows hold `row` and its first row, -1 for none: the last one that
// begins there or before, by a whole warp, 32 ways at a time.
__device__ __forceinline__ int sequence_of_row(const AttnCall& a, int row, int& begin)
{
    const int lane = threadIdx.x & 31;
    int s = -1, high = a.sequences;
    while (high - s > 1)
    {
        const int stride = (high - s + 31) / 32, probe = s + (lane + 1) * stride;
        const int below = __popc(__ballot_sync(0xFFFFFFFFu, probe < high && bounded_offset(a.offsets, probe, a.rows) <= row));
        s += below * stride;
        high = min(high, s + stride);
    }
    if (s < 0)
        return -1;
    begin = bounded_offset(a.offsets, s, a.rows);
    return row < bounded_offset(a.offsets, s + 1, a.rows) ? s : -1;
}

template <bool Tree>
__device__ __forceinline__ RowKeys row_keys(const AttnCall& a, int s, int begin, int row)
{
    RowKeys k;
    k.first = begin;
    k.drafted = row - begin + 1;
    k.cached = 0;
    k.path = ~0ull;
    k.table = nullptr;
    if (Tree)
    {
        k.cached = min(max(a.lengths[s], 0), a.max_length);
        k.path = tree_path(a.parents + begin, row - begin);
        k.table = a.table + (size_t) s * a.table_stride;
    }
    return k;
}

// The weight of a score against the largest so far. Where that is minus infinity every
// score is (or NaN): each weighs 1, so that the sum tells such keys from none at all,
// and drops out as soon as a larger one comes (the sums are scaled by 2^-inf).
__device__ __forceinline__ float weight_of(float score, float m)
{
    return score == -INFINITY && m == -INFINITY ? 1.f : exp2f(score - m);
}

// What a finished row's sums are multiplied with: 0 of a row that attends to nothing,
// NaN where every score is minus infinity and the formula has no weights.
__device__ __forceinline__ float finish_factor(float m, float l)
{
    return l == 0.f ? 0.f : m == -INFINITY ? NAN : 1.f / l;
}

// m, l and the lane's 8 channels of the unnormalised row over keys [from, to)
// of the row's list. All 32 lanes call it.
template <typename T, bool Tree>
__device__ void attend_row(const AttnCall& a, const RowKeys& keys, int kv_head, const float (&q)[8], int from, int to,
                           float& m, float& l, float (&acc)[8])
{
    const int lane = threadIdx.x & 31, c = lane * 8;
    const bool channels = c < a.width;
    const int kvw = a.kv_heads * a.width;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        acc[i] = 0.f;
    for (int base = from; base < to; base += 32)
    {
        // Lane i holds key base + i's rows.
        const int j = base + lane;
        const T* kp = nullptr;
        const T* vp = nullptr;
        if (j < to)
        {
            if (Tree && j < keys.cached)
            {
                const int id = keys.table[j >> kPageLog];
                if (page_there(id, a.pages))
                {
                    const size_t at = ((size_t) id * kPagePositions + (j & (kPagePositions - 1))) * kvw
                                      + (size_t) kv_head * a.width;
                    kp = (const T*) a.key_pages + at;
                    vp = (const T*) a.value_pages + at;
                }
            }
            else if (const int d = j - keys.cached; !Tree || (keys.path >> d & 1))
            {
                kp = (const T*) a.k + (keys.first + d) * a.k_stride + (size_t) kv_head * a.width;
                vp = (const T*) a.v + (keys.first + d) * a.v_stride + (size_t) kv_head * a.width;
            }
        }
        const unsigned seen = __ballot_sync(0xFFFFFFFFu, kp != nullptr);
        if (!seen)
            continue;
        float score = -INFINITY;
        for (unsigned left = seen; left; left &= left - 1)
        {
            const int i = __ffs(left) - 1;
            const T* p = (const T*) __shfl_sync(0xFFFFFFFFu, (unsigned long long) kp, i);
            float dot = 0.f;
            if (channels)
            {
                float x[8];
                load8(p + c, x);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    dot = fmaf(q[e], x[e], dot);
            }
            dot = warp_sum(dot);
            if (lane == i)
                score = dot * a.scale_log2;
        }
        // A NaN score must reach the row: fmaxf drops it, the sums keep it.
        const float m_new = fmaxf(m, warp_max(score));
        const float alpha = m == m_new ? 1.f : exp2f(m - m_new);
        const float weight = kp ? weight_of(score, m_new) : 0.f;
        l = l * alpha + warp_sum(weight);
        float part[8] = {};
        for (unsigned left = seen; left; left &= left - 1)
        {
            const int i = __ffs(left) - 1;
            const T* p = (const T*) __shfl_sync(0xFFFFFFFFu, (unsigned long long) vp, i);
            const float w = __shfl_sync(0xFFFFFFFFu, weight, i);
            if (channels)
            {
                float x[8];
                load8(p + c, x);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    part[e] = fmaf(w, x[e], part[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            acc[e] = fmaf(acc[e], alpha, part[e]);
        m = m_new;
    }
}

// Row `row` (of sequence s, whose rows begin at `begin`), head h, whole.
template <typename T, bool Tree>
__device__ void attention_row(const AttnCall& a, int s, int begin, int row, int h)
{
    const int c = (threadIdx.x & 31) * 8;
    float q[8] = {}, acc[8], m, l;
    if (c < a.width)
        load8((const T*) a.q + row * a.q_stride + (size_t) h * a.width + c, q);
    const RowKeys keys = row_keys<Tree>(a, s, begin, row);
    attend_row<T, Tree>(a, keys, h / a.group, q, 0, keys.cached + keys.drafted, m, l, acc);
    const float inv = finish_factor(m, l);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        acc[e] = l == 0.f ? 0.f : acc[e] * inv;
    if (c < a.width)
        store8((T*) a.out + row * a.out_stride + (size_t) h * a.width + c, acc);
}
} // namespace hfk
