// Attention of packed prompts and drafted trees in fp32 on the 5th-generation
// tensor cores, every operand as two fp16 halves.
//
// Arithmetic. x 2^e = hi + lo with hi = fp16(x 2^e) and lo = fp16(x 2^e - hi) keeps 22
// bits and more of every x that is not tiny next to the largest one under the
// same exponent e, and a product is hi.hi' + hi.lo' + lo.hi' in fp32 (the
// dropped lo.lo' is below 2^-22 of it). The tensor core's fp32 additions
// truncate, so no chain is long at full size: the scores keep hi.hi' (a step
// per 16 channels) and the small rest in accumulators of their own, and the
// values' products of one 64-key tile (the small ones first, then 4 steps of
// hi.hi') are added to the row's fp32 sums in registers, rounded to nearest.
// Exponents: of a query, its row's; of keys and values a tile's (prompts:
// split_tiles takes the tile's largest value) or the CTA's (trees: from 16 of its keys);
// the weights 2^(s - m) are taken times 2^14, which cancels in the end. Where an
// exponent does not fit its tile (rows 2^16 apart; in trees keys or values above some
// 29 to 59 times the sample's largest, or 32 channels of a value below 2^-17 of it) the
// tile's factor is NaN, and like every row that comes out not finite, its rows are
// taken again by attention_row. Rows are looked at, not channels: one whose values are
// all small next to its tile's keeps an error of 2^-39 of the tile's largest value (trees:
// 2^-35 of the sample's), which is more than fp32's below some 2^-20 of it.
//
// Work. As in attention_mma: 128 rows (tokens x a kv head's heads) a unit, 64-key
// tiles, longest rows first, unit after unit. K and V pass through rings of 16 KB
// stages, each 64 keys x 64 channels: the hi half and the lo half. A prompt's keys
// serve many CTAs, so split_tiles writes their halves to the workspace once and the
// stages are tensor-map copies; a tree's keys are read once, so its stages arrive in
// fp32 (the same 16 KB) and a warpgroup of converters turns them into halves in
// place.
//
// Roles: in warpgroup 0 a warp for the copies, one for the scores' MMAs (S = [hi.hi' |
// small] as one MMA of hi with [hi' ; lo'], N = 128, and one of lo with hi', N = 64, a
// step), one for the rows' (three passes of 4 steps over each 64 channels) and one
// that finds places; warpgroups 1 and 2 a row's softmax (half of the keys each) and
// its sums (half of the channels each); in trees warpgroup 3 converts. S is free for
// the next tile once it is in registers; the weights' halves have two buffers.
//
// Measured (B200): 4 x 2048 rows of the engine's heads 263 us, 261 TFLOP/s or 784 in
// fp16 products (0.48 of the measured cuBLAS rate), a tile in some 4,800 cycles where its
// MMAs take 3,330: a tile moves 448 KB through shared memory (128 in, 320 to the
// MMAs), 3,500 cycles of its bandwidth, and at width 256 the queries' halves leave room
// for three stages a ring. In trees the converters bound a tile: about 860 cycles a stage
// (23 cycles a pair of values and warp for the split, 530 for waits and fences).
#pragma once

#include "attention_mma.cuh"

namespace hfk
{
// The two halves of x under a power-of-two factor, two values at a time.
__device__ __forceinline__ void split_pair(float x, float y, float factor, uint32_t& hi, uint32_t& lo)
{
    const float2 v = __fmul2_rn(make_float2(x, y), make_float2(factor, factor));
    const __half2 h = __floats2half2_rn(v.x, v.y);
    const float2 back = __half22float2(h);
    const __half2 l = __floats2half2_rn(v.x - back.x, v.y - back.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// 2^e with `largest` 2^e in [2^top / 2, 2^top); 1 for nothing or for what lies
// outside the normal range by far.
__device__ __forceinline__ float split_factor(float largest, int top)
{
    if (!(largest > 0.f))
        return 1.f;
    const int exponent = (int) (__float_as_uint(largest) >> 23) - 126; // largest in [2^(exponent - 1), 2^exponent)
    const int e = min(max(top - exponent, -120), 120);
    return __uint_as_float((uint32_t) (127 + e) << 23);
}

__device__ __forceinline__ float finite_abs(float x)
{
    const float v = fabsf(x);
    return v < INFINITY ? v : 0.f;
}

struct LimbCall
{
    MmaCall c;
    __half* limbs;    // a prompt's K hi, K lo, V hi, V lo: [4][rows][kv_heads][width]
    float* factors;   // what undoes a tile's exponents: [2][kv_heads][tiles]
    int tiles;        // rows / 64 + sequences: tile j of sequence s is (begin_s / 64) + s + j
};

// One CTA a (tile, kv head, K or V) of packed prompts: 8 rows a warp, 8 channels
// a lane, read once and kept.
__global__ void __launch_bounds__(256) split_tiles(const __grid_constant__ LimbCall l)
{
    __shared__ float row_max[kKeyTile];
    pdl_wait();
    pdl_trigger();
    const AttnCall& a = l.c.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, at = lane * 8;
    const int tile = blockIdx.x, kv_head = blockIdx.y, values = blockIdx.z;
    int low = -1, high = a.sequences; // first(low) <= tile < first(high)
    while (high - low > 1)
    {
        const int mid = (low + high) / 2;
        if (bounded_offset(a.offsets, mid, a.rows) / kKeyTile + mid <= tile)
            low = mid;
        else
            high = mid;
    }
    if (low < 0)
        return;
    const int begin = bounded_offset(a.offsets, low, a.rows);
    const int first = (tile - begin / kKeyTile - low) * kKeyTile;
    const int count = min(bounded_offset(a.offsets, low + 1, a.rows) - begin - first, kKeyTile);
    if (count <= 0)
        return;
    const float* source = (const float*) (values ? a.v : a.k);
    const long long stride = values ? a.v_stride : a.k_stride;
    float x[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const int r = warp * 8 + i;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            x[i][e] = 0.f;
        if (r < count && at < a.width)
            load8(source + (begin + first + r) * stride + (size_t) kv_head * a.width + at, x[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            m = fmaxf(m, finite_abs(x[i][e]));
        m = warp_max(m);
        if (lane == 0)
            row_max[warp * 8 + i] = m;
    }
    __syncthreads();
    const float m0 = row_max[lane], m1 = row_max[lane + 32];
    const float largest = warp_max(fmaxf(m0, m1));
    // The smallest row that counts: of values any, of keys the first that is not
    // zero (a row attends to a tile's keys from the first on).
    const unsigned some0 = __ballot_sync(0xFFFFFFFFu, m0 > 0.f), some1 = __ballot_sync(0xFFFFFFFFu, m1 > 0.f);
    float smallest = -warp_max(-fminf(m0 > 0.f ? m0 : INFINITY, m1 > 0.f ? m1 : INFINITY));
    if (!values && (some0 | some1))
        smallest = row_max[some0 ? __ffs(some0) - 1 : 31 + __ffs(some1)];
    const float factor = split_factor(largest, 15);
    if (tid == 0)
    {
        const bool fits = largest == 0.f || largest * 0x1p-16f <= smallest;
        l.factors[((size_t) values * a.kv_heads + kv_head) * l.tiles + tile] = fits ? 1.f / factor : NAN;
    }
    const size_t limb = (size_t) a.rows * a.kv_heads * a.width;
    if (at < a.width)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            const int r = warp * 8 + i;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                split_pair(x[i][2 * e], x[i][2 * e + 1], factor, hi[e], lo[e]);
            if (r < count)
            {
                __half* to = l.limbs + 2 * values * limb + ((size_t) (begin + first + r) * a.kv_heads + kv_head) * a.width + at;
                *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(to + limb) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
    }
}

template <int D, bool Tree>
struct LimbShape
{
    static constexpr int kBlocks = D / 64;
    static constexpr int kBox = kKeyTile * 128;          // 64 keys x 64 channels of one half
    static constexpr int kStageBytes = 2 * kBox;
    static constexpr int kQueryHalf = kBlocks * 128 * 128;
    static constexpr int kHead = 3 * 1024;
    static constexpr int kStagesFit = (227 * 1024 - kHead - 2 * kQueryHalf) / kStageBytes;
    static constexpr int kStages = kStagesFit > 12 ? 12 : kStagesFit;
    static constexpr int kKeyStages = kStages / 2, kValueStages = kStages - kKeyStages;
    static constexpr int kSmem = kHead + 2 * kQueryHalf + kStages * kStageBytes;
    // O: two buffers, or at width 256 (all that TMEM has left) one in two halves, so
    // that a half is drained while the MMAs fill the other.
    static constexpr int kRowBuffers = D == 256 ? 1 : 2;
    static constexpr bool kHalves = D == 256;
    static constexpr int kThreads = Tree ? 512 : 384;
    // Registers a thread, by warpgroup; at launch 168 or 128 each: the shares
    // add up to that (3 x 168, 4 x 128).
    static constexpr int kLaunchRegisters = Tree ? 128 : 168;
    static constexpr int kRegistersIssue = Tree ? 56 : 72, kRegistersRows = Tree ? 192 : 216, kRegistersConvert = 72;
    static_assert(kRegistersIssue + 2 * kRegistersRows + (Tree ? kRegistersConvert : 0)
                      <= kLaunchRegisters * kThreads / 128,
                  "what the CTA was launched with");
    static constexpr int kScores = 0, kWeights = 128, kRows = 256; // TMEM columns
    static_assert(kRows + kRowBuffers * D <= 512 && kStages >= 6 && kSmem <= 227 * 1024, "what an SM holds");
};

struct LimbHead
{
    uint64_t keys_full[6], keys_ready[6], keys_free[6], values_full[6], values_ready[6], values_free[6];
    uint64_t query, query_free, scores, scores_read, weights[2], done[2], rows_free[2], place_full[2], place_free[2], next,
        sampled[2], drained[2];
    alignas(16) uint4 answer;
    uint32_t tmem;
    int dead;           // a wait ran out
    int misfit[2];         // a unit's value outside its sampled exponent's range
    unsigned sample[2][2]; // a unit's largest sampled K and V, as bits
    MmaPlace place[2];
    int8_t parents[2][kTreeNodes];
};

template <int N>
__device__ __forceinline__ void set_registers_up()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void set_registers_down()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int D, bool Tree>
__global__ void __launch_bounds__(LimbShape<D, Tree>::kThreads, 1)
    attention_limbs(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const __grid_constant__ CUtensorMap kmap2, const __grid_constant__ CUtensorMap vmap2,
                    const __grid_constant__ LimbCall lc)
{
    // Prompts: the maps of K hi, V hi, K lo, V lo. Trees: drafted K, V, paged K, V in fp32.
    using Shape = LimbShape<D, Tree>;
    constexpr int KS = Shape::kKeyStages, VS = Shape::kValueStages, kBlocks = Shape::kBlocks, kHalf = D / 2;
    constexpr int RB = Shape::kRowBuffers;
    extern __shared__ __align__(1024) uint8_t smem[];
    LimbHead& h = *reinterpret_cast<LimbHead*>(smem);
    float(*exchange)[2][128] = reinterpret_cast<float(*)[2][128]>(smem + Shape::kHead - 2048); // [tile parity][warpgroup][row]
    static_assert(sizeof(LimbHead) <= Shape::kHead - 2048, "the head's room");
    uint8_t* queries = smem + Shape::kHead;
    uint8_t* keys = queries + 2 * Shape::kQueryHalf;
    uint8_t* values = keys + KS * Shape::kStageBytes;
    const MmaCall& c = lc.c;
    const AttnCall& a = c.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;

    if (warp == 0 && lane == 0)
    {
        for (int s = 0; s < 6; ++s)
        {
            mbar_init(&h.keys_full[s], 1);
            mbar_init(&h.keys_ready[s], 4); // an arrival a converter warp
            mbar_init(&h.keys_free[s], 1);
            mbar_init(&h.values_full[s], 1);
            mbar_init(&h.values_ready[s], 4);
            mbar_init(&h.values_free[s], 1);
        }
        mbar_init(&h.query, 8); // an arrival a row warp
        mbar_init(&h.query_free, 1);
        mbar_init(&h.scores, 1);
        mbar_init(&h.scores_read, 8);
        mbar_init(&h.next, 1);
        for (int b = 0; b < 2; ++b)
        {
            mbar_init(&h.weights[b], 8);
            mbar_init(&h.done[b], 1);
            mbar_init(&h.rows_free[b], Shape::kHalves ? 4 : 8);
            mbar_init(&h.place_full[b], 1);
            mbar_init(&h.place_free[b], Tree ? 15 : 11); // an arrival a warp but the one that finds them
            mbar_init(&h.drained[b], 1);
            mbar_init(&h.sampled[b], 4); // an arrival a converter warp
        }
        h.dead = 0;
        mbar_fence_init();
    }
    else if (warp == 2 && lane == 0)
    {
        prefetch_map(&kmap);
        prefetch_map(&vmap);
        prefetch_map(&kmap2);
        prefetch_map(&vmap2);
    }
    // Of prompts: split_tiles' halves, of trees whatever is ahead in the stream.
    // TMEM is asked for behind it: that kernel may still want it.
    pdl_wait();
    if (warp == 1)
        tc_alloc(&h.tmem, 512);
    // The first place is found while TMEM is made.
    MmaPlace first = {};
    TreePlaces places;
    if (warp == 3)
    {
        if (Tree)
        {
            places.begin(c, blockIdx.x);
            first = places.next(c);
        }
        else
            first = prompt_place(c, c.tile_tokens, blockIdx.x);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (Tree)
        pdl_trigger(); // attention_join may take its place; it waits for this grid's end
    const uint32_t tmem = h.tmem;
    // A wait of one of the roles; one that runs out ends the CTA's other waits too.
    auto wait = [&](uint64_t* bar, unsigned parity) {
        const bool ok = same_wait(bar, parity);
        if (!ok)
            *(volatile int*) &h.dead = 1;
        return ok;
    };
    // The same where lanes wait for different barriers.
    auto wait_for_all = [&](uint64_t* bar, unsigned parity) {
        const bool ok = warp_wait<2>(bar, parity);
        if (!ok)
            *(volatile int*) &h.dead = 1;
        return ok;
    };
    // The place of the CTA's i-th unit: false when there is none.
    auto take = [&](int i, MmaPlace& p) {
        if (__any_sync(0xFFFFFFFFu, *(volatile int*) &h.dead) || !wait(&h.place_full[i & 1], (i / 2) & 1))
            return false;
        p = h.place[i & 1];
        return p.sequence >= 0;
    };
    auto leave = [&](int i) {
        __syncwarp();
        if (lane == 0)
            mbar_arrive(&h.place_free[i & 1]);
    };
    // Keys of the unit's tile j that are there.
    auto valid_of = [&](const MmaPlace& p, int j) {
        const int t = p.first_tile + j;
        return min(kKeyTile, !Tree                 ? p.length - j * kKeyTile
                             : t < p.tiles_cached ? p.cached - t * kKeyTile
                                                   : p.length);
    };

    if (warp < 4)
    {
        set_registers_down<Shape::kRegistersIssue>();
        if (warp == 0)
        {
            // K and V each in its own order, whichever ring has room: one that waits
            // for its MMAs must not hold up the other (K tile by tile ahead of V,
            // a V that had room came late and a step took 5000 cycles).
            int put_keys = 0, put_values = 0;
            bool ok = true;
            MmaPlace p;
            for (int i = 0; ok && take(i, p); ++i)
            {
                if (lane == 0)
                {
                    const int* table = Tree ? a.table + (size_t) p.sequence * a.table_stride : nullptr;
                    struct
                    {
                        int tile, block, id, id_next;
                    } next[2];
                    auto page_of = [&](int j) {
                        const int t = p.first_tile + j;
                        return Tree && t < p.tiles_cached ? table[t] : -1;
                    };
                    for (int r = 0; r < 2; ++r)
                        next[r] = {0, 0, page_of(0), page_of(1)};
                    auto load = [&](int r, const CUtensorMap* drafted, const CUtensorMap* paged, uint8_t* ring, int& put,
                                    int stages, uint64_t* full, uint64_t* free) {
                        const int stage = put % stages;
                        if (next[r].tile == p.tiles || (put >= stages && !mbar_test(&free[stage], (put / stages - 1) & 1)))
                            return false;
                        const bool cached = Tree && p.first_tile + next[r].tile < p.tiles_cached;
                        const int id = next[r].id, b = next[r].block;
                        // A page that is not there is read past the pool's end: zeros.
                        const int row = cached ? (page_there(id, a.pages) ? id : a.pages) * kPagePositions
                                               : p.begin + (Tree ? 0 : next[r].tile * kKeyTile);
                        uint8_t* to = ring + stage * Shape::kStageBytes;
                        mbar_expect_tx(&full[stage], Shape::kStageBytes);
                        tensor_load(to, Tree && cached ? paged : drafted, 64 * b, p.kv_head, row, &full[stage]);
                        tensor_load(to + Shape::kBox, Tree ? (cached ? paged : drafted) : paged, 64 * b + (Tree ? 32 : 0),
                                    p.kv_head, row, &full[stage]);
                        ++put;
                        if (++next[r].block == kBlocks)
                            next[r] = {next[r].tile + 1, 0, next[r].id_next, page_of(next[r].tile + 2)};
                        return true;
                    };
                    bool idle = false;
                    unsigned begun = 0;
                    while ((next[0].tile < p.tiles || next[1].tile < p.tiles) && ok)
                    {
                        const bool k = load(0, &kmap, &kmap2, keys, put_keys, KS, h.keys_full, h.keys_free);
                        const bool v = load(1, &vmap, &vmap2, values, put_values, VS, h.values_full, h.values_free);
                        const unsigned now = wait_ticks();
                        if (k || v || !idle)
                            begun = now;
                        idle = !k && !v;
                        if (now - begun > kWaitTicks)
                        {
                            flag_error(&g_operator_error, kErrWaitTimeout);
                            *(volatile int*) &h.dead = 1;
                            ok = false;
                        }
                    }
                }
                __syncwarp();
                ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
                leave(i);
            }
            // Every copy has landed before the CTA may end (only a failed run gets here early).
            if (lane == 0 && *(volatile int*) &h.dead)
            {
                for (int n = max(0, put_keys - KS); n < put_keys; ++n)
                    mbar_wait(&h.keys_full[n % KS], (n / KS) & 1);
                for (int n = max(0, put_values - VS); n < put_values; ++n)
                    mbar_wait(&h.values_full[n % VS], (n / VS) & 1);
            }
            __syncwarp();
        }
        else if (warp == 1)
        {
            constexpr uint32_t kWide = tc_idesc16(0, 128, false), kNarrow = tc_idesc16(0, 64, false);
            const uint32_t qhi = smem_addr(queries), qlo = qhi + Shape::kQueryHalf, kbase = smem_addr(keys);
            uint64_t* landed = Tree ? h.keys_ready : h.keys_full;
            int item = 0, count = 0; // stages and tiles before this
            bool ok = true;
            MmaPlace p;
            for (int i = 0; ok && take(i, p); ++i)
            {
                ok = wait(&h.query, i & 1);
                for (int j = 0; j < p.tiles && ok; ++j, ++count)
                {
                    for (int b = 0; b < kBlocks; ++b, ++item)
                    {
                        const int stage = item % KS;
                        const bool reads = (lane & 1) && b == 0 && count > 0; // S of the last tile is in registers
                        ok = wait_for_all(reads ? &h.scores_read : &landed[stage], (reads ? count - 1 : item / KS) & 1);
                        if (!ok)
                            break;
                        tc_fence_after();
                        const uint32_t k = kbase + stage * Shape::kStageBytes;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                        {
                            const uint32_t at = b * 128 * 128 + e * 32;
                            tc_mma_warp(tmem + Shape::kScores, tc_desc(qhi + at), tc_desc(k + e * 32), kWide, b > 0 || e > 0);
                            tc_mma_warp(tmem + Shape::kScores + 64, tc_desc(qlo + at), tc_desc(k + e * 32), kNarrow, 1);
                        }
                        tc_commit_warp(&h.keys_free[stage]);
                    }
                    if (ok)
                        tc_commit_warp(&h.scores);
                }
                if (ok)
                    tc_commit_warp(&h.query_free);
                leave(i);
            }
            finish_mmas(!*(volatile int*) &h.dead, &h.drained[0]);
        }
        else if (warp == 2)
        {
            constexpr uint32_t kValues = tc_idesc16(0, 64, true);
            const uint32_t vbase = smem_addr(values);
            uint64_t* landed = Tree ? h.values_ready : h.values_full;
            int item = 0, count = 0;
            bool ok = true;
            MmaPlace p;
            for (int i = 0; ok && take(i, p); ++i)
            {
                for (int j = 0; j < p.tiles && ok; ++j, ++count)
                {
                    const int valid = valid_of(p, j), buffer = count % RB;
                    for (int b = 0; b < kBlocks; ++b, ++item)
                    {
                        // The stage, the weights, and the buffer's last O in registers.
                        const int stage = item % VS, what = lane & 3, part = Shape::kHalves ? b / 2 : buffer;
                        const bool frees = what == 1 && (b == 0 || (Shape::kHalves && b == 2)) && count >= RB;
                        const bool weighs = what == 2 && b == 0;
                        ok = wait_for_all(frees ? &h.rows_free[part] : weighs ? &h.weights[count & 1] : &landed[stage],
                                          (frees ? count / RB - 1 : weighs ? count / 2 : item / VS) & 1);
                        if (!ok)
                            break;
                        if (!Tree && valid < kKeyTile)
                        {
                            // Rows past the sequence's end: weights of 0, but 0 x NaN is not.
                            const int bytes = (kKeyTile - valid) * 128;
                            for (int box = 0; box < 2; ++box)
                                for (int e = lane * 16; e < bytes; e += 512)
                                    *reinterpret_cast<uint4*>(values + stage * Shape::kStageBytes + box * Shape::kBox
                                                              + valid * 128 + e) = make_uint4(0, 0, 0, 0);
                            fence_proxy_async();
                            __syncwarp();
                        }
                        tc_fence_after();
                        const uint32_t d = tmem + Shape::kRows + buffer * D + b * 64;
                        const uint32_t hi = tmem + Shape::kWeights + (count & 1) * 64, lo = hi + 32;
                        const uint32_t v = vbase + stage * Shape::kStageBytes;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            tc_mma_ts_warp(d, hi + e * 8, tc_desc_mn(v + Shape::kBox + e * 2048, Shape::kBox), kValues, e > 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            tc_mma_ts_warp(d, lo + e * 8, tc_desc_mn(v + e * 2048, Shape::kBox), kValues, 1);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            tc_mma_ts_warp(d, hi + e * 8, tc_desc_mn(v + e * 2048, Shape::kBox), kValues, 1);
                        tc_commit_warp(&h.values_free[stage]);
                        if (b == kBlocks - 1 || (Shape::kHalves && b == 1))
                            tc_commit_warp(&h.done[part]);
                    }
                }
                leave(i);
            }
            finish_mmas(!*(volatile int*) &h.dead, &h.drained[1]);
        }
        else
        {
            // The units' places, found while the unit before is worked on.
            int unit = blockIdx.x, i = 0;
            bool ok = true;
            auto publish = [&](const MmaPlace& p) {
                ok = ok && (i < 2 || wait(&h.place_free[i & 1], (i / 2 - 1) & 1));
                if (ok && lane == 0)
                {
                    h.place[i & 1] = p;
                    mbar_arrive(&h.place_full[i & 1]);
                }
                // The unit's queries on their way to L2 while the one before is worked on.
                if (p.sequence >= 0)
                    for (int t = lane; t < c.tile_tokens && p.token0 + t < p.length; t += 32)
                        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                                         (const float*) a.q + (long long) (p.begin + p.token0 + t) * a.q_stride
                                         + (size_t) p.kv_head * a.group * a.width),
                                     "r"(a.group * a.width * 4)
                                     : "memory");
                ++i;
            };
            if (Tree)
            {
                for (MmaPlace p = first; p.sequence >= 0 && ok; p = places.next(c))
                    publish(p);
            }
            for (int asked = 0; !Tree && ok; ++asked)
            {
                if (lane == 0)
                    ask_next_cta(&h.answer, &h.next);
                const MmaPlace p = asked == 0 ? first : prompt_place(c, c.tile_tokens, unit);
                if (p.sequence >= 0)
                    publish(p);
                ok = wait(&h.next, asked & 1) && ok; // an answer is never left behind
                if (ok && !next_cta(&h.answer, unit))
                    break;
                __syncwarp(); // the answer has been read
            }
            MmaPlace end = {};
            end.sequence = -1; // no more units
            publish(end);
        }
    }
    else if (warp < 12)
    {
        set_registers_up<Shape::kRegistersRows>();
        const int group = (warp - 4) >> 2, quarter = warp & 3;
        const int row = quarter * 32 + lane; // the TMEM lane
        const uint32_t lanes = tmem + ((uint32_t) (quarter * 32) << 16);
        int count = 0; // tiles before this
        // After a wait that ran out a unit goes on without waits, so that the
        // warps' barriers still match.
        bool ok = true;
        MmaPlace p;
        for (int i = 0;; ++i)
        {
            if (any_stops(5, 256, !ok || !take(i, p)))
                break;
            const int tiles = p.tiles;
            const int token = p.token0 + row / a.group, head = p.kv_head * a.group + row % a.group;
            const bool real = row < c.tile_tokens * a.group && token < p.length;
            const bool idle = !__any_sync(0xFFFFFFFFu, real); // no row of the warp's: it keeps the others' step only
            const int* table = Tree ? a.table + (size_t) p.sequence * a.table_stride : nullptr;

            // The queries' halves, a row a warp: lane c the channels [8 c, 8 c + 8).
            ok = ok && (i == 0 || wait(&h.query_free, (i - 1) & 1));
            named_sync(1, 256); // `exchange` is free
#pragma unroll 1
            for (int half = 0; half < 2; ++half)
            {
                float x[8][8];
                int t = ((warp - 4) * 16 + half * 8) / a.group, g = ((warp - 4) * 16 + half * 8) % a.group;
                if (t >= min(c.tile_tokens, p.length - p.token0))
                    break; // rows that are not there may hold anything: it stays with them
                const float* from = (const float*) a.q + (long long) (p.begin + p.token0) * a.q_stride
                                    + (size_t) p.kv_head * a.group * a.width + lane * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        x[e][k] = 0.f;
                    if (t < c.tile_tokens && p.token0 + t < p.length && lane * 8 < a.width)
                        load8(from + t * a.q_stride + (size_t) g * a.width, x[e]);
                    if (++g == a.group)
                        g = 0, ++t;
                }
                // The rows' largest values, eight at once: each step halves the rows that
                // a lane holds, until lanes 4 e .. 4 e + 3 hold row e's (NaN left out; an
                // infinity makes its row NaN, which is what it is).
                float top[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    const float(&v)[8] = x[e];
                    top[e] = max3(max3(max3(0.f, fabsf(v[0]), fabsf(v[1])), fabsf(v[2]), fabsf(v[3])),
                                  max3(0.f, fabsf(v[4]), fabsf(v[5])), max3(0.f, fabsf(v[6]), fabsf(v[7])));
                }
#pragma unroll
                for (int rows = 4; rows >= 1; rows >>= 1)
                {
                    const bool upper = lane & (4 * rows);
#pragma unroll
                    for (int e = 0; e < rows; ++e)
                    {
                        const float other = __shfl_xor_sync(0xFFFFFFFFu, upper ? top[e] : top[e + rows], 4 * rows);
                        top[e] = fmaxf(upper ? top[e + rows] : top[e], other);
                    }
                }
                top[0] = fmaxf(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], 2));
                top[0] = fmaxf(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], 1));
                const float mine = split_factor(top[0], 15);
                if ((lane & 3) == 0)
                    exchange[0][0][(warp - 4) * 16 + half * 8 + lane / 4] = 1.f / mine;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    const int r = (warp - 4) * 16 + half * 8 + e;
                    const float factor = __shfl_sync(0xFFFFFFFFu, mine, 4 * e);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        split_pair(x[e][2 * k], x[e][2 * k + 1], factor, hi[k], lo[k]);
                    if (lane < D / 8)
                    {
                        uint8_t* to = queries + (lane >> 3) * 128 * 128 + r * 128 + (((lane & 7) ^ (r & 7)) << 4);
                        *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4*>(to + Shape::kQueryHalf) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (ok && lane == 0)
                mbar_arrive(&h.query);
            if (Tree)
                for (int e = tid - 128; e < p.length; e += 256)
                    h.parents[i & 1][e] = (int8_t) min(max(a.parents[p.begin + e], -1), kTreeNodes);
            named_sync(1, 256);
            const float row_factor = exchange[0][0][row] * a.scale_log2;
            unsigned path = 0; // of the half's keys
            if (Tree && real)
                path = (unsigned) (tree_path(h.parents[i & 1], token) >> (32 * group));
            const float* kfactors = nullptr;
            const float* vfactors = nullptr;
            float kfactor = 1.f, vfactor = 1.f;
            if (Tree)
            {
                ok = ok && wait(&h.sampled[i & 1], (i / 2) & 1);
                kfactor = 1.f / split_factor(__uint_as_float(h.sample[i & 1][0]), 11);
                vfactor = 1.f / split_factor(__uint_as_float(h.sample[i & 1][1]), 11);
            }
            else
            {
                kfactors = lc.factors + (size_t) p.kv_head * lc.tiles + p.begin / kKeyTile + p.sequence;
                vfactors = kfactors + (size_t) a.kv_heads * lc.tiles;
            }
            named_sync(1, 256); // the row factors have been read

            float acc[kHalf];
#pragma unroll
            for (int e = 0; e < kHalf; ++e)
                acc[e] = 0.f;
            float m = -INFINITY, l = 0.f, alpha_before = 1.f, vfactor_before = 1.f;
            int id = Tree && p.first_tile < p.tiles_cached ? table[p.first_tile] : -1;
            // acc = acc * alpha + (O of the n-th tile) * factor
            auto drain = [&](int n, float alpha, float factor) {
                const int part = Shape::kHalves ? group : n % RB;
                ok = ok && wait(&h.done[part], (n / RB) & 1);
                tc_fence_after();
                const uint32_t at = lanes + Shape::kRows + n % RB * D + group * kHalf;
                const bool scales = __any_sync(0xFFFFFFFFu, alpha != 1.f);
#pragma unroll
                for (int b = 0; b < kHalf; b += 32)
                {
                    if (idle)
                        break;
                    uint32_t o[32];
                    tc_ld32(at + b, o);
                    tc_wait_ld32(o);
                    if (scales)
                    {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            acc[b + e] *= alpha;
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        acc[b + e] = fmaf(__uint_as_float(o[e]), factor, acc[b + e]);
                }
                tc_fence_before();
                __syncwarp();
                if (ok && lane == 0)
                    mbar_arrive(&h.rows_free[part]);
            };
            for (int j = 0; j < tiles; ++j, ++count)
            {
                const int t = p.first_tile + j;
                const int id_next = Tree && t + 1 < p.tiles_cached ? table[t + 1] : -1;
                if (!Tree)
                {
                    kfactor = kfactors[j];
                    vfactor = vfactors[j];
                }
                // S is there. The weights' buffer is free: the MMAs that read it two
                // tiles back ended before O of that tile was drained, by both
                // warpgroups before the last tile's exchange.
                ok = ok && wait(&h.scores, count & 1);
                tc_fence_after();
                if (idle)
                {
                    if (ok && lane == 0)
                    {
                        mbar_arrive(&h.scores_read);
                        mbar_arrive(&h.weights[count & 1]);
                    }
                    named_sync(1, 256);
                    if (j > 0)
                        drain(count - 1, 1.f, 0.f);
                    continue;
                }
                float s[32];
                {
                    uint32_t large[32], small[32];
                    tc_ld32(lanes + Shape::kScores + group * 32, large);
                    tc_ld32(lanes + Shape::kScores + 64 + group * 32, small);
                    tc_wait_ld32(large);
                    tc_wait_ld32(small);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        s[e] = __uint_as_float(large[e]) + __uint_as_float(small[e]);
                }
                tc_fence_before();
                __syncwarp();
                if (ok && lane == 0)
                    mbar_arrive(&h.scores_read);
                // What the row does not attend to.
                if (Tree && t >= p.tiles_cached)
                {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        s[e] = path >> e & 1 ? s[e] : -INFINITY;
                }
                else
                {
                    const int limit = (!Tree                        ? token - j * kKeyTile + 1
                                       : page_there(id, a.pages) ? p.cached - t * kKeyTile
                                                                  : 0)
                                      - 32 * group;
                    if (limit < 32)
                    {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            s[e] = e < limit ? s[e] : -INFINITY;
                    }
                }
                id = id_next;
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int e = 4; e < 28; e += 8)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        top[g] = max3(top[g], s[e + 2 * g], s[e + 2 * g + 1]);
                const float mine = max3(max3(top[0], s[28], s[29]), max3(top[1], s[30], s[31]), fmaxf(top[2], top[3]));
                exchange[j & 1][group][row] = mine;
                named_sync(1, 256);
                const float factor = row_factor * kfactor;
                const float m_new = fmaxf(m, fmaxf(mine, exchange[j & 1][group ^ 1][row]) * factor);
                const float alpha = m == m_new ? 1.f : exp2_approx(m - m_new);
                const float base = 14.f - (m_new == -INFINITY ? 0.f : m_new);
                m = m_new;
                float2 sum[2] = {};
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int e = 0; e < 16; ++e)
                {
                    const float2 x = __ffma2_rn(make_float2(s[2 * e], s[2 * e + 1]), make_float2(factor, factor),
                                                make_float2(base, base));
                    const float2 w = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                    sum[e & 1] = __fadd2_rn(sum[e & 1], w);
                    const __half2 hh = __floats2half2_rn(w.x, w.y);
                    const float2 back = __half22float2(hh);
                    hi[e] = *reinterpret_cast<const uint32_t*>(&hh);
                    lo[e] = pack_pair<__half>(w.x - back.x, w.y - back.y);
                }
                l = l * alpha + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
                const uint32_t wbase = lanes + Shape::kWeights + (count & 1) * 64 + group * 16;
                tc_st16(wbase, hi);
                tc_st16(wbase + 32, lo);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (ok && lane == 0)
                    mbar_arrive(&h.weights[count & 1]);
                if (j > 0)
                    drain(count - 1, alpha_before, vfactor_before);
                alpha_before = alpha;
                vfactor_before = vfactor;
            }
            drain(count - 1, alpha_before, vfactor_before);
            exchange[tiles & 1][group][row] = l;
            named_sync(1, 256);
            l += exchange[tiles & 1][group ^ 1][row];
            const bool whole = !Tree || p.whole;
            const int at = p.begin + token;
            const size_t part = (size_t) p.part * c.part_rows + row;
            // The weights' 2^14: cancels in a finished row, is taken off a part's.
            const float scaled = !ok ? NAN : l == 0.f ? 0.f : whole ? 1.f / l : 0x1p-14f;
            // 0 for finite values. A maximum of minus infinity may be of masked keys or of such scores.
            float2 check = make_float2(l * 0.f, m == -INFINITY || (Tree && *(volatile int*) &h.misfit[i & 1]) ? NAN : 0.f);
            char* mine = (char*) (whole ? (float*) a.out + at * a.out_stride + (size_t) head * a.width
                                        : c.part_o + part * a.width);
            // Through the queries' room (their last MMA is over): a row a thread in,
            // a row a warp out, 16-byte chunk c of row r at chunk c ^ r.
            constexpr int kChunks = kHalf / 4;
            float4* room = reinterpret_cast<float4*>(queries) + (warp - 4) * 32 * kChunks;
#pragma unroll
            for (int b = 0; b < kChunks; ++b)
            {
                if (idle)
                    break;
                float2 v[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                {
                    v[e] = make_float2(acc[4 * b + 2 * e], acc[4 * b + 2 * e + 1]);
                    check = __ffma2_rn(v[e], make_float2(0.f, 0.f), check);
                    v[e] = __fmul2_rn(v[e], make_float2(scaled, scaled));
                }
                room[lane * kChunks + (b ^ lane & (kChunks - 1))] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
            }
            __syncwarp();
            const unsigned rows = __ballot_sync(0xFFFFFFFFu, real);
            constexpr int kAtOnce = 32 / kChunks; // rows
            const int chunk = lane & (kChunks - 1), channel = group * kHalf + 4 * chunk;
#pragma unroll 4
            for (int r0 = 0; r0 < 32 && !idle; r0 += kAtOnce)
            {
                const int r = r0 + lane / kChunks;
                char* to = (char*) __shfl_sync(0xFFFFFFFFu, (unsigned long long) mine, r);
                if (rows >> r & 1 && channel < a.width)
                    *reinterpret_cast<float4*>(to + 4 * channel) = room[r * kChunks + (chunk ^ r & (kChunks - 1))];
            }
            if (Tree && !whole && real && group == 0)
                c.part_ml[part] = make_float2(m, l * 0x1p-14f);
            if (Tree && real && group == 0 && p.first_tile == 0 && row % a.group == 0)
                c.spans[(size_t) at * a.kv_heads + p.kv_head] = span_of(p, blockIdx.x);
            const bool finite = check.x + check.y == 0.f;
            exchange[(tiles & 1) ^ 1][group][row] = finite ? 0.f : 1.f;
            named_sync(1, 256);
            // Rows that came out not finite: again, half of them by each warpgroup's warp.
            unsigned again = __ballot_sync(0xFFFFFFFFu, ok && real && (!finite || exchange[(tiles & 1) ^ 1][group ^ 1][row] != 0.f));
            again &= group ? 0xAAAAAAAAu : 0x55555555u;
            while (again)
            {
                const int who = __ffs(again) - 1;
                again &= again - 1;
                take_again<float, Tree>(c, h.place[i & 1], __shfl_sync(0xFFFFFFFFu, at, who), __shfl_sync(0xFFFFFFFFu, head, who));
            }
            leave(i);
        }
        tc_fence_before();
    }
    else if (Tree)
    {
        set_registers_down<Shape::kRegistersConvert>();
        const int t = tid - 384;
        // A stage: thread t holds 32 channels (one fp32 box's row) of key t / 2.
        const int key = t >> 1, box = t & 1;
        int taken_keys = 0, taken_values = 0;
        bool ok = true; // as with the row warps
        MmaPlace p;
        for (int i = 0;; ++i)
        {
            if (any_stops(2, 128, !ok || !take(i, p)))
                break;
            const int tiles = p.tiles;
            const int* table = a.table + (size_t) p.sequence * a.table_stride;
            // The exponents: the largest of 16 keys spread over the unit's, an
            // eighth of their channels a thread. The row warps have left the unit
            // before the last, whose slot this is.
            if (t < 2)
                h.sample[i & 1][t] = 0;
            if (t == 2)
                h.misfit[i & 1] = 0;
            named_sync(3, 128);
            {
                const int end = min((p.first_tile + tiles) * kKeyTile, p.cached), from = p.first_tile * kKeyTile;
                const int which = t >> 3;
                const float* k = nullptr;
                const float* v = nullptr;
                if (end > from)
                {
                    const int j = from + (int) ((long long) (end - from) * which / 16);
                    const int page = table[j >> kPageLog];
                    if (page_there(page, a.pages))
                    {
                        const size_t at = (((size_t) page << kPageLog) + (j & (kPagePositions - 1))) * a.kv_heads + p.kv_head;
                        k = (const float*) a.key_pages + at * a.width;
                        v = (const float*) a.value_pages + at * a.width;
                    }
                }
                else
                {
                    const int r = p.begin + p.length * which / 16;
                    k = (const float*) a.k + r * a.k_stride + (size_t) p.kv_head * a.width;
                    v = (const float*) a.v + r * a.v_stride + (size_t) p.kv_head * a.width;
                }
                float mk = 0.f, mv = 0.f;
                for (int e = (t & 7) * 4; k && e < a.width; e += 32)
                {
                    const float4 x = *reinterpret_cast<const float4*>(k + e), y = *reinterpret_cast<const float4*>(v + e);
                    mk = fmaxf(fmaxf(mk, fmaxf(finite_abs(x.x), finite_abs(x.y))), fmaxf(finite_abs(x.z), finite_abs(x.w)));
                    mv = fmaxf(fmaxf(mv, fmaxf(finite_abs(y.x), finite_abs(y.y))), fmaxf(finite_abs(y.z), finite_abs(y.w)));
                }
                mk = warp_max(mk), mv = warp_max(mv);
                if (lane == 0)
                {
                    atomicMax(&h.sample[i & 1][0], __float_as_uint(mk));
                    atomicMax(&h.sample[i & 1][1], __float_as_uint(mv));
                }
            }
            named_sync(3, 128);
            const float factors[2] = {split_factor(__uint_as_float(h.sample[i & 1][0]), 11),
                                      split_factor(__uint_as_float(h.sample[i & 1][1]), 11)};
            if (lane == 0)
                mbar_arrive(&h.sampled[i & 1]);
            bool misfit = false;
            auto convert = [&](int j, float factor, bool is_value, uint8_t* ring, int& taken, int stages, uint64_t* full,
                               uint64_t* ready) {
                const bool there = key < valid_of(p, j);
                for (int b = 0; b < kBlocks; ++b)
                {
                    const int stage = taken % stages;
                    ok = ok && wait(&full[stage], (taken / stages) & 1);
                    uint8_t* at = ring + stage * Shape::kStageBytes + key * 128;
                    uint32_t hi[16], lo[16];
                    float largest = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                    {
                        float4 x = *reinterpret_cast<const float4*>(at + box * Shape::kBox + ((e ^ (key & 7)) << 4));
                        if (!there)
                            x = make_float4(0.f, 0.f, 0.f, 0.f); // behind the sequence: whatever the page holds
                        largest = fmaxf(fmaxf(largest, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
                        split_pair(x.x, x.y, factor, hi[2 * e], lo[2 * e]);
                        split_pair(x.z, x.w, factor, hi[2 * e + 1], lo[2 * e + 1]);
                    }
                    // Too large for fp16, or values so small that their halves lose digits.
                    largest *= factor;
                    misfit = misfit || largest > 60000.f || (is_value && largest > 0.f && largest < 0x1p-6f);
                    named_sync(3, 128); // all of the stage's fp32 is in registers
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                    {
                        const int chunk = ((box * 4 + e) ^ (key & 7)) << 4;
                        *reinterpret_cast<uint4*>(at + chunk) =
                            make_uint4(hi[4 * e], hi[4 * e + 1], hi[4 * e + 2], hi[4 * e + 3]);
                        *reinterpret_cast<uint4*>(at + Shape::kBox + chunk) =
                            make_uint4(lo[4 * e], lo[4 * e + 1], lo[4 * e + 2], lo[4 * e + 3]);
                    }
                    if (misfit)
                        *(volatile int*) &h.misfit[i & 1] = 1;
                    fence_proxy_async();
                    __syncwarp();
                    if (ok && lane == 0)
                        mbar_arrive(&ready[stage]);
                    ++taken;
                }
            };
            for (int j = 0; j <= tiles; ++j)
            {
                if (j < tiles)
                    convert(j, factors[0], false, keys, taken_keys, KS, h.keys_full, h.keys_ready);
                if (j > 0)
                    convert(j - 1, factors[1], true, values, taken_values, VS, h.values_full, h.values_ready);
            }
            leave(i);
        }
    }
    __syncthreads();
    if (warp == 1)
        tc_dealloc(tmem, 512);
}
} // namespace hfk
