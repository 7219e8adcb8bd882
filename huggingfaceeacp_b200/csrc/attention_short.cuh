// Attention of the smallest calls: a CTA a (row, head), its keys cut for four warps
// (attend_short), whose maxima, sums and rows meet in shared memory. One launch with
// no copies to set up and no parts to join, where the tiled kernels' set-up would
// be most of the call. What bounds it is latency: offsets, lengths, pages, keys and
// values, one read after another. Eight keys a warp in flight: with four, one row of
// 100 keys takes 12.6 us instead of 10.4. is_short in operators.cu says which calls come
// here, and what they take.
#pragma once

#include "attention_rows.cuh"

namespace hfk
{
constexpr int kShortWarps = 4, kShortKeys = 8;

// attend_row with the loads of kShortKeys keys in flight. (The tiled kernels, which call
// attend_row for the rows that they take again, have no registers for this one: with it
// a call for 64 caches of 4000 took 204 us instead of 188.)
template <typename T, bool Tree>
__device__ __forceinline__ void attend_short(const AttnCall& a, const RowKeys& keys, int kv_head, const float (&q)[8],
                                             int from, int to, float& m, float& l, float (&acc)[8])
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
        for (unsigned left = seen; left;)
        {
            int who[kShortKeys]; // -1: no key left
            float x[kShortKeys][8];
#pragma unroll
            for (int n = 0; n < kShortKeys; ++n)
            {
                who[n] = __ffs(left) - 1;
                left &= left - 1;
                const T* p = (const T*) __shfl_sync(0xFFFFFFFFu, (unsigned long long) kp, max(who[n], 0));
                if (channels && who[n] >= 0)
                    load8(p + c, x[n]);
            }
#pragma unroll
            for (int n = 0; n < kShortKeys; ++n)
            {
                float dot = 0.f;
                if (channels && who[n] >= 0)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        dot = fmaf(q[e], x[n][e], dot);
                dot = warp_sum(dot);
                if (lane == who[n])
                    score = dot * a.scale_log2;
            }
        }
        // A NaN score must reach the row: fmaxf drops it, the sums keep it.
        const float m_new = fmaxf(m, warp_max(score));
        const float alpha = m == m_new ? 1.f : exp2f(m - m_new);
        const float weight = kp ? weight_of(score, m_new) : 0.f;
        l = l * alpha + warp_sum(weight);
        float part[8] = {};
        for (unsigned left = seen; left;)
        {
            int who[kShortKeys];
            float x[kShortKeys][8];
#pragma unroll
            for (int n = 0; n < kShortKeys; ++n)
            {
                who[n] = __ffs(left) - 1;
                left &= left - 1;
                const T* p = (const T*) __shfl_sync(0xFFFFFFFFu, (unsigned long long) vp, max(who[n], 0));
                if (channels && who[n] >= 0)
                    load8(p + c, x[n]);
            }
#pragma unroll
            for (int n = 0; n < kShortKeys; ++n)
            {
                const float w = __shfl_sync(0xFFFFFFFFu, weight, max(who[n], 0));
                if (channels && who[n] >= 0)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        part[e] = fmaf(w, x[n][e], part[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            acc[e] = fmaf(acc[e], alpha, part[e]);
        m = m_new;
    }
}

template <typename T, bool Tree>
__global__ void __launch_bounds__(32 * kShortWarps, 4) attention_short(const __grid_constant__ AttnCall a)
{
    __shared__ float rows[kShortWarps][256];
    __shared__ float2 sums[kShortWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, at = lane * 8;
    const int row = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
    float q[8] = {}, acc[8], m, l;
    pdl_wait();
    pdl_trigger();
    if (at < a.width)
        load8((const T*) a.q + row * a.q_stride + (size_t) head * a.width + at, q);
    int begin;
    const int s = sequence_of_row(a, row, begin);
    if (s < 0 || (Tree && row - begin >= a.max_nodes))
        return; // the CTA together
    const RowKeys keys = row_keys<Tree>(a, s, begin, row);
    const int count = keys.cached + keys.drafted, share = (count + kShortWarps - 1) / kShortWarps;
    attend_short<T, Tree>(a, keys, head / a.group, q, min(warp * share, count), min((warp + 1) * share, count), m, l, acc);
    store8(&rows[warp][at], acc);
    if (lane == 0)
        sums[warp] = make_float2(m, l);
    __syncthreads();
    if (warp)
        return;
    // A part in which nothing was attended weighs nothing; of none, the row is 0.
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kShortWarps; ++w)
        m = fmaxf(m, sums[w].y == 0.f ? -INFINITY : sums[w].x);
    l = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kShortWarps; ++w)
    {
        if (sums[w].y == 0.f)
            continue;
        const float weight = sums[w].x == m ? 1.f : exp2f(sums[w].x - m);
        float x[8];
        load8(&rows[w][at], x);
        l = fmaf(weight, sums[w].y, l);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            acc[e] = fmaf(weight, x[e], acc[e]);
    }
    const float inv = finish_factor(m, l);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        acc[e] = l == 0.f ? 0.f : acc[e] * inv;
    if (at < a.width)
        store8((T*) a.out + row * a.out_stride + (size_t) head * a.width + at, acc);
}
} // namespace hfk
