// Attention of drafted trees over a paged cache in fp32 where a kv head has at most
// eight query rows (an ordinary decode step of the engine's eight heads, a tree
// of two nodes over four, ...): plain fp32 FMAs.
//
// A cached position is read once and meets 8 rows, 4 operations for each 4 bytes and
// row: about 3,200 issue slots a scheduler and 64-key tile at width 256 against the
// 5,400 cycles that the tile takes to arrive at 44 GB/s an SM. Measured (B200), 64
// sequences of 200 to 2,048 tokens, the engine's heads: 47 us a call for 122 MB, a tile
// in 6,300 cycles, the rest its start, the warps' meeting and the join.
// (attention_limbs, whose converters take 8,000 cycles a tile: 91 us.)
//
// Work. The key tiles are shared out to the CTAs as for the other trees. Tiles pass
// through a ring in halves of 32 keys, K then V, each one tensor-map copy; warp w
// takes keys 4 w to 4 w + 3 of each. A lane holds 4 channels of every 128: the sums of
// all eight rows in registers, the queries in shared memory (nine warps get 168
// registers each), so that rows are read by conflict-free 16-byte loads. The 4 x 8
// scores are summed over the lanes by halving (31 shuffles: lane r + 8 k ends with row r,
// key k). Each warp has its own running maximum and sum over its own keys, and its
// own rows of O; the warps meet at the end of a unit. No fp32 chain is longer than a
// warp's keys.
#pragma once

#include "attention_mma.cuh"

namespace hfk
{
constexpr int kFewRows = 8;
constexpr int kFewWarps = 8;
constexpr int kFewKeys = 32; // of a stage

template <int D>
struct FewShape
{
    static constexpr int kVectors = (D + 127) / 128; // 4-channel pieces a lane
    static constexpr int kStageBytes = kFewKeys * D * 4;
    static constexpr int kHead = 1024;
    static constexpr int kMeet = kFewWarps * kFewRows * (D + 2) * 4; // the warps' rows at the end of a unit
    static constexpr int kStages = D == 256 ? 4 : 8;
    static constexpr int kQueries = kFewRows * D * 4;
    static constexpr int kSmem = kHead + kMeet + kQueries + kStages * kStageBytes;
    static constexpr int kThreads = 32 * (kFewWarps + 1);
    static_assert(kSmem <= 227 * 1024 && kStages % 4 == 0, "what an SM holds; a unit's items begin at any stage");
};

struct FewHead
{
    uint64_t full[8], empty[8], place_full[2], place_free[2];
    int dead; // a wait ran out
    MmaPlace place[2];
};

template <int D>
__global__ void __launch_bounds__(FewShape<D>::kThreads, 1)
    attention_few(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                  const __grid_constant__ CUtensorMap kpages, const __grid_constant__ CUtensorMap vpages,
                  const __grid_constant__ MmaCall c)
{
    using Shape = FewShape<D>;
    constexpr int S = Shape::kStages, V = Shape::kVectors;
    extern __shared__ __align__(1024) uint8_t smem[];
    FewHead& h = *reinterpret_cast<FewHead*>(smem);
    static_assert(sizeof(FewHead) <= Shape::kHead, "the head's room");
    uint8_t* ring = smem + Shape::kHead;
    float4* queries = reinterpret_cast<float4*>(ring + S * Shape::kStageBytes); // [row][channel]
    float* meet = reinterpret_cast<float*>(ring + S * Shape::kStageBytes + Shape::kQueries);
    const AttnCall& a = c.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;

    if (tid == 0)
    {
        for (int s = 0; s < S; ++s)
        {
            mbar_init(&h.full[s], 1);
            mbar_init(&h.empty[s], kFewWarps);
        }
        for (int b = 0; b < 2; ++b)
        {
            mbar_init(&h.place_full[b], 1);
            mbar_init(&h.place_free[b], kFewWarps);
        }
        h.dead = 0;
        mbar_fence_init();
    }
    else if (tid == 32)
    {
        prefetch_map(&kmap);
        prefetch_map(&vmap);
        prefetch_map(&kpages);
        prefetch_map(&vpages);
    }
    pdl_wait();
    __syncthreads();
    pdl_trigger(); // attention_join may take its place; it waits for this grid's end

    if (warp == kFewWarps)
    {
        TreePlaces places;
        places.begin(c, blockIdx.x);
        int put = 0;
        bool ok = true;
        auto one_wait = [&](uint64_t* bar, unsigned parity) {
            if (ok && !lone_wait(bar, parity))
            {
                *(volatile int*) &h.dead = 1;
                ok = false;
            }
            return ok;
        };
        for (int i = 0;; ++i)
        {
            const MmaPlace p = places.next(c);
            if (lane == 0 && (i < 2 || one_wait(&h.place_free[i & 1], (i / 2 - 1) & 1)))
            {
                h.place[i & 1] = p;
                mbar_arrive(&h.place_full[i & 1]);
            }
            ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
            if (p.sequence < 0 || !ok)
                break;
            const int* table = a.table + (size_t) p.sequence * a.table_stride;
            int ids = -1; // 32 tiles' pages
            for (int j = 0; j < p.tiles; ++j)
            {
                const int t = p.first_tile + j;
                if ((j & 31) == 0)
                    ids = t + lane < p.tiles_cached ? table[t + lane] : -1;
                const int id = __shfl_sync(0xFFFFFFFFu, ids, j & 31);
                if (lane == 0)
                {
                    const bool cached = t < p.tiles_cached;
                    // A page that is not there is read past the pool's end: zeros.
                    const int row = cached ? (page_there(id, a.pages) ? id : a.pages) * kPagePositions : p.begin;
                    for (int part = 0; part < 4; ++part) // K and V of the first 32 keys, then of the others
                    {
                        const int stage = put % S;
                        if (put >= S && !one_wait(&h.empty[stage], (put / S - 1) & 1))
                            break;
                        mbar_expect_tx(&h.full[stage], Shape::kStageBytes);
                        tensor_load(ring + stage * Shape::kStageBytes,
                                    part & 1 ? (cached ? &vpages : &vmap) : (cached ? &kpages : &kmap), 0, p.kv_head,
                                    row + part / 2 * kFewKeys, &h.full[stage]);
                        ++put;
                    }
                }
                __syncwarp();
            }
        }
        // Every copy has landed before the CTA may end (only a failed run gets here early).
        if (lane == 0 && !ok)
            for (int n = max(0, put - S); n < put; ++n)
                mbar_wait(&h.full[n % S], (n / S) & 1);
        __syncwarp();
        return;
    }

    // Lane r + 8 k: row r, key k of the warp's four.
    const int row = lane & 7, key = lane >> 3;
    int item = 0;
    bool ok = true; // after a wait that ran out the CTA goes on without waits, so that its barriers still match
    for (int i = 0;; ++i)
    {
        const bool come = ok && !__any_sync(0xFFFFFFFFu, *(volatile int*) &h.dead)
                          && same_wait(&h.place_full[i & 1], (i / 2) & 1);
        if (any_stops(1, 32 * kFewWarps, !come || h.place[i & 1].sequence < 0))
            break;
        const MmaPlace p = h.place[i & 1];
        const int* table = a.table + (size_t) p.sequence * a.table_stride;
        const int rows = min(p.length - p.token0, c.tile_tokens) * a.group; // at most eight
        float4 acc[kFewRows][V];
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v)
                acc[r][v] = make_float4(0.f, 0.f, 0.f, 0.f);
        // A row a warp; the warps' meeting at the end of the last unit freed the room.
#pragma unroll
        for (int v = 0; v < V; ++v)
        {
            const int channel = 128 * v + 4 * lane, token = p.begin + p.token0 + warp / a.group;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (warp < rows && channel < a.width)
                x = *reinterpret_cast<const float4*>((const float*) a.q + token * a.q_stride
                                                     + (size_t) (p.kv_head * a.group + warp % a.group) * a.width + channel);
            if (channel < D)
                queries[warp * (D / 4) + 32 * v + lane] = x;
        }
        named_sync(2, 32 * kFewWarps);
        unsigned long long path = 0;
        if (row < rows)
            path = tree_path(a.parents + p.begin, p.token0 + row / a.group);
        float m = -INFINITY, l = 0.f; // of the lane's row, over the warp's keys; l of the lane's key only
        for (int j = 0; j < p.tiles; ++j)
        {
            const int t = p.first_tile + j;
            const bool cached = t < p.tiles_cached;
            const int valid = cached ? (page_there(table[t], a.pages) ? min(kPagePositions, p.cached - t * kKeyTile) : 0) : p.length;
#pragma unroll 1
            for (int half = 0; half < 2; ++half, item += 2)
            {
                const int first = half * kFewKeys + 4 * warp; // the warp's keys of the tile
                const int ks = item % S, vs = (item + 1) % S;
                ok = ok && same_wait(&h.full[ks], (item / S) & 1);
                float s[4 * kFewRows];
                {
                    float4 x[4][V];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int v = 0; v < V; ++v)
                            x[k][v] = 128 * v + 4 * lane < D
                                          ? reinterpret_cast<const float4*>(ring + ks * Shape::kStageBytes
                                                                            + (4 * warp + k) * D * 4)[32 * v + lane]
                                          : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int r = 0; r < kFewRows; ++r)
                    {
                        float dot[4] = {};
#pragma unroll
                        for (int v = 0; v < V; ++v)
                        {
                            const float4 q = 128 * v + 4 * lane < D ? queries[r * (D / 4) + 32 * v + lane]
                                                                    : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                            {
                                dot[k] = fmaf(q.x, x[k][v].x, dot[k]);
                                dot[k] = fmaf(q.y, x[k][v].y, dot[k]);
                                dot[k] = fmaf(q.z, x[k][v].z, dot[k]);
                                dot[k] = fmaf(q.w, x[k][v].w, dot[k]);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            s[8 * k + r] = dot[k];
                    }
                }
                __syncwarp();
                if (ok && lane == 0)
                    mbar_arrive(&h.empty[ks]);
                // Sum over the lanes: at each step a lane keeps the half of the scores
                // that its bit names.
#pragma unroll
                for (int n = 16; n >= 1; n >>= 1)
                {
                    const bool upper = lane & n;
#pragma unroll
                    for (int e = 0; e < n; ++e)
                    {
                        const float other = __shfl_xor_sync(0xFFFFFFFFu, upper ? s[e] : s[e + n], n);
                        s[e] = (upper ? s[e + n] : s[e]) + other;
                    }
                }
                const int mine = first + key;
                const bool seen = row < rows && mine < valid && (cached || (path >> mine & 1));
                const float score = seen ? s[0] * a.scale_log2 : -INFINITY;
                // fmaxf leaves a NaN score out; its weight brings it back.
                float m_new = fmaxf(m, score);
                m_new = fmaxf(m_new, __shfl_xor_sync(0xFFFFFFFFu, m_new, 8));
                m_new = fmaxf(m_new, __shfl_xor_sync(0xFFFFFFFFu, m_new, 16));
                const float alpha = m == m_new ? 1.f : exp2_approx(m - m_new);
                const float weight = seen && score != -INFINITY ? exp2_approx(score - m_new) : 0.f;
                l = l * alpha + weight;
                m = m_new;
                if (__any_sync(0xFFFFFFFFu, alpha != 1.f))
                {
#pragma unroll
                    for (int r = 0; r < kFewRows; ++r)
                    {
                        const float scale = __shfl_sync(0xFFFFFFFFu, alpha, r);
#pragma unroll
                        for (int v = 0; v < V; ++v)
                            acc[r][v] = make_float4(acc[r][v].x * scale, acc[r][v].y * scale, acc[r][v].z * scale,
                                                    acc[r][v].w * scale);
                    }
                }
                ok = ok && same_wait(&h.full[vs], ((item + 1) / S) & 1);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                {
                    if (first + k < valid) // a row behind the sequence may hold anything
                    {
                        const float4* from =
                            reinterpret_cast<const float4*>(ring + vs * Shape::kStageBytes + (4 * warp + k) * D * 4);
                        float4 x[V];
#pragma unroll
                        for (int v = 0; v < V; ++v)
                            x[v] = 128 * v + 4 * lane < D ? from[32 * v + lane] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int r = 0; r < kFewRows; ++r)
                        {
                            const float w = __shfl_sync(0xFFFFFFFFu, weight, r + 8 * k);
#pragma unroll
                            for (int v = 0; v < V; ++v)
                            {
                                acc[r][v].x = fmaf(w, x[v].x, acc[r][v].x);
                                acc[r][v].y = fmaf(w, x[v].y, acc[r][v].y);
                                acc[r][v].z = fmaf(w, x[v].z, acc[r][v].z);
                                acc[r][v].w = fmaf(w, x[v].w, acc[r][v].w);
                            }
                        }
                    }
                }
                __syncwarp();
                if (ok && lane == 0)
                    mbar_arrive(&h.empty[vs]);
            }
        }
        // The warps meet: each leaves its rows, maxima and sums, then takes one row.
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 8);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
        named_sync(2, 32 * kFewWarps); // the last unit's rows have been taken
        float* mine = meet + warp * kFewRows * (D + 2);
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (128 * v + 4 * lane < D)
                {
                    float2* to = reinterpret_cast<float2*>(mine + r * (D + 2) + 128 * v + 4 * lane);
                    to[0] = make_float2(acc[r][v].x, acc[r][v].y);
                    to[1] = make_float2(acc[r][v].z, acc[r][v].w);
                }
        if (lane < kFewRows)
        {
            mine[lane * (D + 2) + D] = m;
            mine[lane * (D + 2) + D + 1] = l;
        }
        named_sync(2, 32 * kFewWarps);
        if (warp < rows)
        {
            const float* from = meet + warp * (D + 2);
            constexpr int kStep = kFewRows * (D + 2); // from warp to warp
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w)
                top = fmaxf(top, from[w * kStep + D]);
            float weight[kFewWarps];
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w)
            {
                const float lw = from[w * kStep + D + 1], mw = from[w * kStep + D];
                weight[w] = lw == 0.f ? 0.f : mw == top ? 1.f : exp2f(mw - top);
                sum += weight[w] * lw;
            }
            const int at = p.begin + p.token0 + warp / a.group, head = p.kv_head * a.group + warp % a.group;
            const size_t part = (size_t) p.part * c.part_rows + warp;
            const float scaled = !ok ? NAN : sum == 0.f ? 0.f : p.whole ? 1.f / sum : 1.f;
            float* to = p.whole ? (float*) a.out + at * a.out_stride + (size_t) head * a.width : c.part_o + part * a.width;
            // Stays 0 for finite values. A maximum of minus infinity may be of masked keys or of such scores.
            float check = top == -INFINITY ? NAN : sum * 0.f;
            for (int channel = 2 * lane; channel < a.width; channel += 64)
            {
                float2 x = make_float2(0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kFewWarps; ++w)
                {
                    const float2 y = *reinterpret_cast<const float2*>(from + w * kStep + channel);
                    check = fmaf(y.x + y.y, 0.f, check);
                    x.x = fmaf(weight[w], y.x, x.x);
                    x.y = fmaf(weight[w], y.y, x.y);
                }
                *reinterpret_cast<float2*>(to + channel) = make_float2(x.x * scaled, x.y * scaled);
            }
            if (!p.whole && lane == 0)
                c.part_ml[part] = make_float2(top, sum);
            if (p.first_tile == 0 && warp % a.group == 0 && lane == 0)
                c.spans[(size_t) at * a.kv_heads + p.kv_head] = span_of(p, blockIdx.x);
            __syncwarp();
            if (__any_sync(0xFFFFFFFFu, ok && !(check == 0.f)))
                take_again<float, true>(c, h.place[i & 1], at, head);
        }
        __syncwarp();
        if (lane == 0)
            mbar_arrive(&h.place_free[i & 1]);
    }
}
} // namespace hfk
