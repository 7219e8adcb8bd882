// Attention of the smallest calls: a CTA a (row, head), its keys cut for four warps
// (attend_row), whose maxima, sums and rows meet in shared memory. One launch with
// no copies to set up and no parts to join, where the tiled kernels' set-up would
// be most of the call. What bounds it is latency: offsets, lengths, pages, keys and
// values, one read after another. Eight keys a warp in flight: with four, one row of
// 100 keys takes 12.6 us instead of 10.4. is_short in operators.cu says which calls come
// here, and what they take.
#pragma once

#include "attention_rows.cuh"

namespace hfk
{
constexpr int kShortWarps = 4;

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
    // The row's sequence: the last one that begins at the row or before it, 32 ways at a time.
    int s = -1, high = a.sequences;
    while (high - s > 1)
    {
        const int stride = (high - s + 31) / 32, probe = s + (lane + 1) * stride;
        const int below = __popc(__ballot_sync(0xFFFFFFFFu, probe < high && bounded_offset(a.offsets, probe, a.rows) <= row));
        s += below * stride;
        high = min(high, s + stride);
    }
    if (s < 0 || row >= bounded_offset(a.offsets, s + 1, a.rows))
        return; // the CTA together
    const int begin = bounded_offset(a.offsets, s, a.rows);
    if (Tree && row - begin >= a.max_nodes)
        return;
    const RowKeys keys = row_keys<Tree>(a, s, begin, row);
    const int count = keys.cached + keys.drafted, share = (count + kShortWarps - 1) / kShortWarps;
    attend_row<T, Tree, 8>(a, keys, head / a.group, q, min(warp * share, count), min((warp + 1) * share, count), m, l, acc);
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
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        acc[e] = l == 0.f ? 0.f : acc[e] * inv;
    if (at < a.width)
        store8((T*) a.out + row * a.out_stride + (size_t) head * a.width + at, acc);
}
} // namespace hfk
