// Attention of packed prompts and drafted trees in bf16 and fp16 on the
// 5th-generation tensor cores: scores S = Q K^T and rows O = P V as
// tcgen05.mma with fp32 accumulators in TMEM, one pass over the keys with the
// running maximum and sum of a softmax.
//
// Work. A query tile is 128 rows: `tile_tokens` consecutive tokens x the heads
// that share one kv head (row = token * group + head), so short prompts and
// single tokens fill it as far as they can and a causal tile's ragged edge is
// a few tokens wide. A CTA takes NQ query tiles of one kv head, over the same
// keys, in tiles of 64 (a page).
//
// Roles:
//  places   a warp finds the next unit while this one is worked on;
//  copies   query tiles, then key and value tiles, each through a ring of its
//           own (tensor maps; a page is one box), on into the next unit as far
//           as there is room. (Of one ring for both, a warp that takes only the
//           keys would see every other phase of a stage's barrier, and its parity
//           cannot tell a phase from the one two before.)
//  MMAs     a warp for each query tile's S and one for its O, since a warp's
//           waits and MMAs follow one another: S of the next tile is issued as
//           soon as S of this one is in registers, O of a tile as soon as its
//           weights are in TMEM;
//  softmax  a warpgroup a query tile, a thread a row (its TMEM lane): the tile's
//           scores to registers, maximum, weights, the weights in T back to TMEM
//           in one of two buffers (P, the A operand of O += P V), at the end
//           the row itself.
// A CTA takes unit after unit. Of prompts, it cancels the launch of a CTA that has not
// started and does its work (the order stays the grid's, longest rows first), so
// that the next unit's copies and scores run under this one's last steps.
// The maximum that the weights are taken against follows the true one lazily:
// only when it would rise by more than 8 (weights up to 2^8) is O scaled in
// TMEM, which after the first tiles is rare. Weights are rounded to T for the
// tensor core (half a step relative to each), their sum is kept in fp32
// unrounded.
//
// Value rows past a sequence's last key are set to zero in shared memory before
// the MMA (their weights are 0, but 0 x NaN is not). Inside a sequence a
// masked value that is not finite makes the tile's sums NaN for rows that do not
// attend to it: every row that comes out not finite, or has a score of NaN or
// infinity, is taken again by attention_row, which reads only what the row attends to.
//
// A batch of trees is shared out evenly in key tiles, so a query tile's keys may
// lie with several CTAs: each leaves its rows' maximum, sum and unnormalised O in
// the workspace, and attention_join puts them together.
//
// Measured (B200, CUDA events). Prompts, 4 x 4096 tokens, 32 heads of 128 over 8:
// 510 us, 1,075 TFLOP/s, 0.65 of the measured cuBLAS rate, the tensor pipe active
// 52 % of the time; 8 heads of 256 over one: 1,212 TFLOP/s, 59 %. Bound by the
// softmax warps: a step of both query tiles (256 rows x 64 keys) takes some 1,700
// cycles, 1,000 of them the weights, whose special-function (640), FMA (540) and
// ALU (580) time two warps a scheduler overlap only partly; its MMAs take 1,280
// (N = 64 scores are bound by the 6 KB that each reads from shared memory, 48
// cycles instead of 32). Tried and no faster: two warpgroups a query tile, the
// tiles' warps taking turns, 2 or 4 of 8 pairs on the FMA pipe. Trees, one token for
// each of 64 caches of 4,000: 163 us in this kernel (profiled alone) for 1.07 GB, 1.0 of
// the measured copy rate; the call, with attention_join and its start, 189.
#pragma once

#include "attention_rows.cuh"
#include "key_span.cuh"
#include "phases.cuh"
#include "tcgen05.cuh"

namespace hfk
{
constexpr int kKeyTile = 64;
static_assert(kKeyTile == kPagePositions, "a key tile is a page");

// Set when a bounded wait ran out (hf_cuda_operators_sync reports it).
__device__ unsigned g_operator_error;

struct MmaCall
{
    AttnCall a;
    int tile_tokens; // tokens of a query tile: 128 / group
    int ctas;        // a tree's: its key tiles are shared out to that many
    int start;       // a tree's: what a unit's start and end cost, in key tiles
    int part_rows;   // rows of a part: a query tile's at most
    float* part_o;   // [2 ctas][part_rows][width]
    float2* part_ml; // [2 ctas][part_rows]
    int2* spans;     // [rows][kv_heads]: the first and the last CTA that hold a row's keys (few: first | kFew)
};

// 2^x of two values on the FMA pipe: x = n + f with n the nearest integer (the
// addition of 1.5 2^23 leaves it in the low bits), 2^f on [-1/2, 1/2] by the
// polynomial of least largest relative error (Remez exchange; 7.5e-5 at degree
// 3, 2.6e-6 at degree 4), n added to the exponent. Below 2^-126 it returns about
// that, where exp2_approx gives 0, and for NaN too: its callers look for NaN in the
// scores' maximum.
template <int Degree>
__device__ __forceinline__ float2 exp2_poly(float2 x)
{
    constexpr float kMagic = 12582912.f;
    x.x = fmaxf(x.x, -126.f);
    x.y = fmaxf(x.y, -126.f);
    const float2 t = __fadd2_rn(x, make_float2(kMagic, kMagic));
    const float2 n = __fadd2_rn(t, make_float2(-kMagic, -kMagic));
    const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
    constexpr float c3[] = {0.9999280571937561f, 0.6932609677314758f, 0.2426111251115799f, 0.0551716685295105f};
    constexpr float c4[] = {0.9999992847442627f, 0.6931217908859253f, 0.240247443318367f, 0.05591785907745361f,
                            0.009570102207362652f};
    const float* c = Degree == 3 ? c3 : c4;
    float2 p = make_float2(c[Degree], c[Degree]);
#pragma unroll
    for (int i = Degree - 1; i >= 0; --i)
        p = __ffma2_rn(p, f, make_float2(c[i], c[i]));
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                       __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}

// The tile's 64 scores of a row to weights 2^(s scale + base), packed in T, and
// their sum. The special-function unit makes 16 values of 2^x a cycle and SM,
// which at head width 128 takes as long as the MMAs; of a tile without masked
// scores (`Mixed`) kPoly of 8 pairs go to the FMA pipe instead.
template <typename T, bool Mixed>
__device__ __forceinline__ float weigh(const float* s, float scale, float base, uint32_t* w)
{
    constexpr int kPoly = 3, kDegree = std::is_same<T, __nv_bfloat16>::value ? 3 : 4;
    float2 sum[2] = {};
#pragma unroll
    for (int i = 0; i < 32; ++i)
    {
        const float2 x = __ffma2_rn(make_float2(s[2 * i], s[2 * i + 1]), make_float2(scale, scale),
                                    make_float2(base, base));
        const float2 e = Mixed && i % 8 * kPoly % 8 < kPoly ? exp2_poly<kDegree>(x)
                                                           : make_float2(exp2_approx(x.x), exp2_approx(x.y));
        sum[i & 1] = __fadd2_rn(sum[i & 1], e);
        w[i] = pack_pair<T>(e.x, e.y);
    }
    return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
}

template <int D, int NQ>
struct MmaShape
{
    static constexpr int kBlocks = D / 64;                 // 64-channel blocks of a row
    static constexpr int kQueryBytes = NQ * 128 * D * 2;
    static constexpr int kStageBytes = kKeyTile * D * 2;   // one K or V tile
    static constexpr int kBox = kKeyTile * 128;            // one block of it
    static constexpr int kScoreColumns = NQ * 2 * kKeyTile; // a query tile's scores and two buffers of weights
    static constexpr int kTmem = kScoreColumns + NQ * D <= 256 ? 256 : 512;
    static constexpr int kCtas = kTmem == 256 ? 2 : 1;     // a SM
    static constexpr int kHead = 2048;                     // barriers, places
    static constexpr int kBudget = kCtas == 2 ? 113 * 1024 : 227 * 1024;
    static constexpr int kStagesFit = (kBudget - kHead - kQueryBytes) / kStageBytes;
    static constexpr int kStages = kStagesFit > 12 ? 12 : kStagesFit;
    static constexpr int kKeyStages = kStages / 2, kValueStages = kStages - kKeyStages;
    static constexpr int kSmem = kHead + kQueryBytes + kStages * kStageBytes;
    static constexpr int kThreads = 128 + 128 * NQ + (NQ == 2 ? 64 : 0); // the last warps: MMAs, places
    static_assert(kScoreColumns + NQ * D <= kTmem && kStages >= 4, "what an SM holds");
};

// A unit's place.
struct MmaPlace
{
    int sequence; // -1: nothing to do; published: no more units
    int begin, length; // its first row, its rows (a tree's nodes)
    int token0, kv_head, part;
    int cached, tiles_cached; // a tree's
    int first_tile, tiles;    // its key tiles
    int last_cta;             // a tree's that begins here: who holds its last tile
    bool few;
    bool whole;               // all of its keys: finish the rows
};

struct MmaHead
{
    uint64_t keys_full[6], keys_free[6], values_full[6], values_free[6], query, query_free, scores[2], scores_read[2], weights[2][2], done[2][2], rows_free[2],
        place_full[2], place_free[2], next, drained[4];
    alignas(16) uint4 answer;
    uint32_t tmem;
    int dead; // a wait ran out
    MmaPlace place[2];
    int parents[2][kTreeNodes];
};

// Bounded waits, of a warp together and of one thread. A warp's lanes may name
// different barriers: it goes on when all have come, for the price of one.
//
// The limit is in time: the hardware holds a poll that finds nothing for 4 us while all
// of a warp's lanes wait, and for 0.09 us once some have gone on, so that a number of
// polls says little. After 8 to 9 ticks of 2^32 ns, some 36 s, a wait gives up: far
// above a step, and above the rows that a warp may have to take again meanwhile, at
// 0.43 us a key and row (32 rows of two million keys; in attention_limbs 16 at 0.52).
// Where it is known how the lanes wait, polls are counted: same_wait, of a warp whose
// lanes all wait for one barrier (34 s), and lone_wait, of one thread (24 s).
//
// The loop has one way on and one out: with a second way on (a slower loop behind it, a
// call, a look at whether rows are taken again) the compiler no longer sees that the
// lanes go together, and calls take 5 to 60 % longer. The clock is read after every
// `Polls`, which decides between a wait's length and the code's. Measured with 1, 2, 4
// and 8: prompts of 32 heads of 128, 4 x 4096 tokens 515, 509, 509, 513 us, 2048 of up to
// 64 tokens 307, 295, 262, 274; of width 256 479, 464, 464, 452; 2048 decode steps of 10 to
// 600 tokens 878, 886, 926, 1014, one tree of 63 14.7, 14.9, 15.9, 15.5. (48 fp32 decode
// steps on FMAs: 94.6, 95.2, 95.6, 95.6, with counted polls 93.3.)
#ifndef HFK_WAIT_TICKS // a test shortens it
#define HFK_WAIT_TICKS 8
#endif
constexpr unsigned kWaitTicks = HFK_WAIT_TICKS;

__device__ __forceinline__ unsigned wait_ticks()
{
    unsigned t;
    asm volatile("mov.u32 %0, %%globaltimer_hi;" : "=r"(t));
    return t;
}

template <int Polls>
__device__ __forceinline__ bool timed_wait(uint64_t* bar, unsigned parity)
{
    unsigned begun = 0;
    for (bool first = true;; first = false)
    {
#pragma unroll
        for (int i = 0; i < Polls; ++i)
            if (mbar_wait(bar, parity, 1))
                return true;
        const unsigned now = wait_ticks();
        if (first)
            begun = now;
        if (now - begun > kWaitTicks)
            return false;
    }
}
template <int Polls>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, unsigned parity)
{
    if (__all_sync(0xFFFFFFFFu, timed_wait<Polls>(bar, parity)))
        return true;
    flag_error(&g_operator_error, kErrWaitTimeout);
    return false;
}
template <int Polls>
__device__ __forceinline__ bool thread_wait(uint64_t* bar, unsigned parity)
{
    if (timed_wait<Polls>(bar, parity))
        return true;
    flag_error(&g_operator_error, kErrWaitTimeout);
    return false;
}
__device__ __forceinline__ bool same_wait(uint64_t* bar, unsigned parity)
{
    if (__all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, 1u << 23)))
        return true;
    flag_error(&g_operator_error, kErrWaitTimeout);
    return false;
}
__device__ __forceinline__ bool lone_wait(uint64_t* bar, unsigned parity)
{
    if (mbar_wait(bar, parity, 1u << 28))
        return true;
    flag_error(&g_operator_error, kErrWaitTimeout);
    return false;
}

// The sequences' tiles of `step` tokens in descending order of their place (the
// longest rows of keys first), equal places in the sequences' order: unit r of
// them, by a whole warp. A lane keeps the tile counts of its sequences (lane, lane
// + 32, ...) in registers; past kKnown of them it reads the offsets again.
__device__ inline void find_tile(const AttnCall& a, int step, int r, int& sequence, int& tile)
{
    constexpr int kKnown = 4;
    const int lane = threadIdx.x & 31;
    auto tiles_of = [&](int s) {
        if (s >= a.sequences)
            return 0;
        const int n = bounded_offset(a.offsets, s + 1, a.rows) - bounded_offset(a.offsets, s, a.rows);
        return n > 0 ? (n + step - 1) / step : 0;
    };
    int known[kKnown], most = 0;
#pragma unroll
    for (int i = 0; i < kKnown; ++i)
        most = max(most, known[i] = tiles_of(lane + 32 * i));
    for (int s = lane + 32 * kKnown; s < a.sequences; s += 32)
        most = max(most, tiles_of(s));
    auto from = [&](int t) { // tiles whose place is t or above
        int sum = 0;
#pragma unroll
        for (int i = 0; i < kKnown; ++i)
            sum += max(known[i] - t, 0);
        for (int s = lane + 32 * kKnown; s < a.sequences; s += 32)
            sum += max(tiles_of(s) - t, 0);
        return __reduce_add_sync(0xFFFFFFFFu, sum);
    };
    int low = 0, high = __reduce_max_sync(0xFFFFFFFFu, most); // from(low) > r >= from(high)
    sequence = -1;
    if (from(0) <= r)
        return;
    while (high - low > 1)
    {
        const int mid = (low + high) / 2;
        if (from(mid) > r)
            low = mid;
        else
            high = mid;
    }
    tile = low;
    int skip = r - from(low + 1);
    for (int i = 0; 32 * i < a.sequences; ++i)
    {
        const int mine = i == 0 ? known[0] : i == 1 ? known[1] : i == 2 ? known[2] : i == 3 ? known[3] : tiles_of(lane + 32 * i);
        unsigned has = __ballot_sync(0xFFFFFFFFu, mine > low);
        const int n = __popc(has);
        if (skip < n)
        {
            while (skip--)
                has &= has - 1;
            sequence = 32 * i + __ffs(has) - 1;
            return;
        }
        skip -= n;
    }
}

// The same of more sequences than a lane keeps, in the sequences' order, each one's
// last tile first: tile j of sequence s has number begin_s / step + s + j, so a search
// 32 ways at a time finds it (in descending order of place each unit would cost a
// pass over all sequences).
__device__ inline void find_tile_of_many(const AttnCall& a, int step, int r, int& sequence, int& tile)
{
    const int lane = threadIdx.x & 31;
    int low = -1, high = a.sequences; // the number of low's first tile <= r < that of high's
    while (high - low > 1)
    {
        const int stride = (high - low + 31) / 32, s = low + (lane + 1) * stride;
        const bool below = s < high && bounded_offset(a.offsets, s, a.rows) / step + s <= r;
        const int n = __popc(__ballot_sync(0xFFFFFFFFu, below));
        low += n * stride;
        high = min(high, low + stride);
    }
    sequence = -1;
    if (low < 0)
        return;
    const int begin = bounded_offset(a.offsets, low, a.rows);
    const int length = bounded_offset(a.offsets, low + 1, a.rows) - begin, tiles = (length + step - 1) / step;
    tile = tiles - 1 - (r - begin / step - low);
    if (length > 0 && tile >= 0)
        sequence = low;
}

// Where unit `unit` (a CTA of the grid) of packed prompts works, its rows in steps
// of `step` tokens; by a whole warp.
__device__ inline MmaPlace prompt_place(const MmaCall& c, int step, int unit)
{
    const AttnCall& a = c.a;
    MmaPlace p = {};
    int s, tile = 0;
    p.kv_head = unit % a.kv_heads;
    if (a.sequences <= 128)
        find_tile(a, step, unit / a.kv_heads, s, tile);
    else
        find_tile_of_many(a, step, unit / a.kv_heads, s, tile);
    p.sequence = s;
    if (s >= 0)
    {
        p.begin = bounded_offset(a.offsets, s, a.rows);
        p.length = bounded_offset(a.offsets, s + 1, a.rows) - p.begin;
        p.token0 = tile * step;
        p.tiles = (min(p.token0 + step, p.length) - 1) / kKeyTile + 1;
        p.whole = true;
    }
    return p;
}

// A batch of trees is one row of key tiles: sequence after sequence, in it query tile
// after query tile of each kv head, of each its cached tiles and the drafted one.
// It is cut for the CTAs in one of two ways:
//  few query tiles (a CTA's share is less than a quarter of one): each is cut into pieces
//  of at most `per` tiles, no more pieces than CTAs. A CTA takes one piece: a
//  second would cost it another start (about 10 us of a 60 us call of 16 trees in
//  fp32);
//  many: every CTA takes `per` tiles in a row, whatever query tiles they fall on, so
//  that sequences of any lengths keep all CTAs busy to the end. Each query tile is
//  preceded by `start` tiles that nobody reads: what it costs to begin and to end.
// A query tile that a CTA holds whole is finished there; of one that several share, each
// leaves a part: part 2 cta + 1 where the query tile begins in a row of many, else 2 cta.
// The host refuses calls of 2^30 tiles and more.
struct TreeRow
{
    int nodes, cached, tiles, query_tiles; // of a sequence; tiles a query tile
    __device__ int total() const { return tiles * query_tiles; }
};

__device__ __forceinline__ TreeRow tree_row(const MmaCall& c, int s)
{
    const AttnCall& a = c.a;
    TreeRow r = {};
    if (s >= a.sequences)
        return r;
    const int begin = bounded_offset(a.offsets, s, a.rows);
    r.nodes = max(min(bounded_offset(a.offsets, s + 1, a.rows) - begin, a.max_nodes), 0);
    r.cached = min(max(a.lengths[s], 0), a.max_length);
    r.tiles = (r.cached + kKeyTile - 1) / kKeyTile + 1;
    r.query_tiles = (r.nodes + c.tile_tokens - 1) / c.tile_tokens * a.kv_heads;
    return r;
}

struct TreeCut
{
    bool few;
    int per;
    __device__ int pieces(int tiles) const { return (tiles + per - 1) / per; } // few: of a query tile
};

// How a call's row is cut, and its tiles; by a whole warp, `known` the lane's of the
// first 32 sequences. At least two tiles a CTA: a part costs about one.
__device__ inline TreeCut cut_trees(const MmaCall& c, const TreeRow& known, int& total)
{
    const int lane = threadIdx.x & 31, sequences = c.a.sequences;
    total = known.total();
    int query_tiles = known.query_tiles;
    for (int s = lane + 32; s < sequences; s += 32)
    {
        const TreeRow r = tree_row(c, s);
        total += r.total();
        query_tiles += r.query_tiles;
    }
    total = __reduce_add_sync(0xFFFFFFFFu, total);
    query_tiles = __reduce_add_sync(0xFFFFFFFFu, query_tiles);
    // The sum of n / per, each rounded up, is at most total / per + query_tiles.
    const bool few = 4 * query_tiles <= c.ctas;
    const int share = few ? c.ctas - query_tiles : c.ctas;
    if (!few)
        total += c.start * query_tiles;
    return {few, max((total + share - 1) / share, 2)};
}

// The places of CTA `cta` one after another; by a whole warp.
struct TreePlaces
{
    TreeRow known; // the lane's of the first 32 sequences
    TreeCut cut;
    int at, end, cta;       // tiles; few: pieces
    int base = 0, before = 0; // the 32 sequences to go on from, and what lies before them

    __device__ void begin(const MmaCall& c, int which)
    {
        int total;
        cta = which;
        known = tree_row(c, threadIdx.x & 31);
        cut = cut_trees(c, known, total);
        at = cut.few ? cta : min(total, cta * cut.per);
        end = cut.few ? cta + 1 : min(total, at + cut.per);
    }
    // A sequence's tiles, or pieces, in the row.
    __device__ int share(const MmaCall& c, const TreeRow& r) const
    {
        return r.query_tiles * (cut.few ? cut.pieces(r.tiles) : r.tiles + c.start);
    }
    __device__ MmaPlace next(const MmaCall& c)
    {
        const AttnCall& a = c.a;
        const int lane = threadIdx.x & 31;
        MmaPlace p = {};
        p.sequence = -1;
        for (; base < a.sequences && at < end; base += 32)
        {
            const TreeRow mine = base ? tree_row(c, base + lane) : known;
            int sum = share(c, mine);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1)
            {
                const int up = __shfl_up_sync(0xFFFFFFFFu, sum, o);
                if (lane >= o)
                    sum += up;
            }
            const unsigned beyond = __ballot_sync(0xFFFFFFFFu, before + sum > at);
            if (beyond)
            {
                const int who = __ffs(beyond) - 1;
                const int within = at - before - __shfl_sync(0xFFFFFFFFu, sum - share(c, mine), who);
                const int tiles = __shfl_sync(0xFFFFFFFFu, mine.tiles, who), each = cut.few ? cut.pieces(tiles) : tiles + c.start;
                const int query_tile = within / each, rest = within - query_tile * each;
                p.sequence = base + who;
                p.begin = bounded_offset(a.offsets, p.sequence, a.rows);
                p.length = __shfl_sync(0xFFFFFFFFu, mine.nodes, who);
                p.cached = __shfl_sync(0xFFFFFFFFu, mine.cached, who);
                p.tiles_cached = tiles - 1;
                p.kv_head = query_tile % a.kv_heads;
                p.token0 = query_tile / a.kv_heads * c.tile_tokens;
                if (cut.few) // pieces as even as they go
                {
                    p.first_tile = (int) ((long long) tiles * rest / each);
                    p.tiles = (int) ((long long) tiles * (rest + 1) / each) - p.first_tile;
                    p.part = 2 * cta;
                    p.last_cta = cta + each - 1;
                    p.few = true;
                    at = end;
                }
                else
                {
                    const int begin = at - rest; // the query tile's place in the row
                    p.first_tile = max(rest - c.start, 0);
                    p.tiles = min(each, end - begin) - c.start - p.first_tile;
                    p.part = 2 * cta + (p.first_tile == 0);
                    p.last_cta = (begin + each - 1) / cut.per; // where first_tile is 0
                    at = min(begin + each, end);
                    if (p.tiles <= 0) // the CTA ends before its first key tile
                        p.sequence = -1;
                }
                p.whole = p.tiles == tiles;
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, sum, 31);
        }
        return p;
    }
};

// What a unit that begins its query tile leaves for attention_join.
__device__ __forceinline__ int2 span_of(const MmaPlace& p, int cta)
{
    return make_int2(p.few ? cta | kFew : cta, p.last_cta);
}

// A row that came out not finite, by a whole warp: the same keys again, read
// only where the row attends to them.
template <typename T, bool Tree>
__device__ __noinline__ void take_again(const MmaCall& c, const MmaPlace& p, int row, int head)
{
    const AttnCall& a = c.a;
    if (!Tree || p.whole)
    {
        attention_row<T, Tree>(a, p.sequence, p.begin, row, head);
        return;
    }
    const int at = (threadIdx.x & 31) * 8;
    const RowKeys keys = row_keys<Tree>(a, p.sequence, p.begin, row);
    const int from = min(p.first_tile * kKeyTile, keys.cached), end = p.first_tile + p.tiles;
    const int to = end > p.tiles_cached ? keys.cached + keys.drafted : min(end * kKeyTile, keys.cached);
    float q[8] = {}, acc[8], m, l;
    if (at < a.width)
        load8((const T*) a.q + row * a.q_stride + (size_t) head * a.width + at, q);
    attend_row<T, Tree>(a, keys, p.kv_head, q, from, to, m, l, acc);
    const size_t part = (size_t) p.part * c.part_rows + (row - p.begin - p.token0) * a.group + head % a.group;
    if (at < a.width)
        store8(c.part_o + part * a.width + at, acc);
    if (at == 0)
        c.part_ml[part] = make_float2(m, l);
}

__device__ __forceinline__ void named_sync(int id, int threads)
{
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Whether any of the barrier's threads wants to stop: warps that share barriers leave
// their loops together.
__device__ __forceinline__ bool any_stops(int id, int threads, bool stop)
{
    uint32_t any;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n barrier.cta.red.or.aligned.pred q, %1, %2, p;\n"
                 " selp.u32 %0, 1, 0, q;\n}"
                 : "=r"(any)
                 : "r"(id), "r"(threads), "r"((uint32_t) stop)
                 : "memory");
    return any;
}

// A failed run: the MMAs that the warp has issued end before TMEM is given back.
__device__ __forceinline__ void finish_mmas(bool ok, uint64_t* bar)
{
    if (!ok)
    {
        tc_commit_warp(bar);
        mbar_wait(bar, 0);
    }
}

// Four lanes' 64 bytes each (four rows, 16 registers a lane as chunks of 4) to four
// chunks of 64 bytes a row: lane i of the four ends with chunk i of rows 0 to 3,
// so that a store of chunk k writes 64 consecutive bytes of a row.
__device__ __forceinline__ void turn4(uint32_t (&r)[16])
{
    const int lane = threadIdx.x & 3;
#pragma unroll
    for (int bit = 1; bit <= 2; bit <<= 1)
#pragma unroll
        for (int c = 0; c < 4; ++c)
        {
            if (c & bit)
                continue;
            const bool upper = lane & bit;
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                uint32_t& low = r[4 * c + i];
                uint32_t& high = r[4 * (c | bit) + i];
                const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, upper ? low : high, bit);
                (upper ? low : high) = got;
            }
        }
}

// The 16 registers (64 bytes) of each lane's row to `to` + 64 bytes * block, the
// lanes' rows where `real`, bytes from `end` on left out. `rows`: four lanes' pointers.
__device__ __forceinline__ void store_rows(uint32_t (&r)[16], char* const (&rows)[4], unsigned real, int at, int end)
{
    turn4(r);
    const int lane = threadIdx.x & 31;
    at += (lane & 3) * 16;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (real >> ((lane & ~3) + k) & 1 && at < end)
            *reinterpret_cast<uint4*>(rows[k] + at) = make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
}

template <typename T, int D, int NQ, bool Tree>
__global__ void __launch_bounds__(MmaShape<D, NQ>::kThreads, MmaShape<D, NQ>::kCtas)
    attention_mma(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap kpages,
                  const __grid_constant__ CUtensorMap vpages, const __grid_constant__ MmaCall c)
{
    using Shape = MmaShape<D, NQ>;
    constexpr int KS = Shape::kKeyStages, VS = Shape::kValueStages, kBlocks = Shape::kBlocks;
    constexpr int kType = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    constexpr int kPolls = Tree ? 1 : D == 256 ? 8 : 4; // see timed_wait
    extern __shared__ __align__(1024) uint8_t smem[];
    MmaHead& h = *reinterpret_cast<MmaHead*>(smem);
    static_assert(sizeof(MmaHead) <= Shape::kHead, "the head's room");
    uint8_t* queries = smem + Shape::kHead;
    uint8_t* keys = queries + Shape::kQueryBytes;
    uint8_t* values = keys + KS * Shape::kStageBytes;
    const AttnCall& a = c.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;

    if (warp == 0 && lane == 0)
    {
        for (int s = 0; s < KS; ++s)
        {
            mbar_init(&h.keys_full[s], 1);
            mbar_init(&h.keys_free[s], NQ); // an arrival an MMA warp
        }
        for (int s = 0; s < VS; ++s)
        {
            mbar_init(&h.values_full[s], 1);
            mbar_init(&h.values_free[s], NQ);
        }
        mbar_init(&h.query, 1);
        mbar_init(&h.query_free, NQ);
        mbar_init(&h.next, 1);
        for (int b = 0; b < 2; ++b)
        {
            mbar_init(&h.place_full[b], 1);
            mbar_init(&h.place_free[b], 6 * NQ + 1); // an arrival a warp but the one that finds them
        }
        for (int q = 0; q < NQ; ++q)
        {
            mbar_init(&h.scores[q], 1);
            mbar_init(&h.scores_read[q], 4); // an arrival a warp
            mbar_init(&h.rows_free[q], 4);
            mbar_init(&h.drained[q], 1);
            mbar_init(&h.drained[2 + q], 1);
            for (int b = 0; b < 2; ++b)
            {
                mbar_init(&h.weights[q][b], 4);
                mbar_init(&h.done[q][b], 1);
            }
        }
        h.dead = 0;
        mbar_fence_init();
    }
    else if (warp == 2 && lane == 0)
    {
        prefetch_map(&qmap);
        prefetch_map(&kmap);
        prefetch_map(&vmap);
        if (Tree)
        {
            prefetch_map(&kpages);
            prefetch_map(&vpages);
        }
    }
    // The set-up above ran beside the end of the kernel ahead in the stream. TMEM is
    // asked for behind it: that kernel may still want it.
    pdl_wait();
    if (warp == 1)
        tc_alloc(&h.tmem, Shape::kTmem);
    // The first place is found while TMEM is made.
    MmaPlace first = {};
    TreePlaces places;
    if (warp == (NQ == 2 ? 13 : 3))
    {
        if (Tree)
        {
            places.begin(c, blockIdx.x);
            first = places.next(c);
        }
        else
            first = prompt_place(c, c.tile_tokens * NQ, blockIdx.x);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (Tree)
        pdl_trigger(); // attention_join may take its place; it waits for this grid's end
    const uint32_t tmem = h.tmem;
    // Key tiles of query tile q: a prompt's tile ends with its last token's.
    auto tiles_of = [&](const MmaPlace& p, int q) {
        const int t0 = p.token0 + q * c.tile_tokens;
        if (t0 >= p.length)
            return 0;
        return Tree ? p.tiles : (min(t0 + c.tile_tokens, p.length) - 1) / kKeyTile + 1;
    };
    // A wait of one of the roles; one that runs out ends the CTA's other waits too.
    auto wait = [&](uint64_t* bar, unsigned parity) {
        const bool ok = warp_wait<kPolls>(bar, parity);
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

    if (warp == 0)
    {
        int put_keys = 0, put_values = 0, put_queries = 0;
        bool ok = true;
        auto one_wait = [&](uint64_t* bar, unsigned parity) {
            if (ok && !thread_wait<kPolls>(bar, parity))
            {
                *(volatile int*) &h.dead = 1;
                ok = false;
            }
            return ok;
        };
        MmaPlace p;
        for (int i = 0; ok && take(i, p); ++i)
        {
            const int tiles = p.tiles;
            const int* table = Tree ? a.table + (size_t) p.sequence * a.table_stride : nullptr;
            auto load = [&](int j, const CUtensorMap* drafted, const CUtensorMap* paged, int id, uint8_t* ring, int& put,
                            int stages, uint64_t* full, uint64_t* free) {
                const int stage = put % stages;
                if (!ok || (put >= stages && !one_wait(&free[stage], (put / stages - 1) & 1)))
                    return;
                const bool cached = Tree && p.first_tile + j < p.tiles_cached;
                // A page that is not there is read past the pool's end: zeros.
                const int row = cached ? (page_there(id, a.pages) ? id : a.pages) * kPagePositions
                                       : p.begin + (Tree ? 0 : j * kKeyTile);
                mbar_expect_tx(&full[stage], Shape::kStageBytes);
                for (int b = 0; b < kBlocks; ++b)
                    tensor_load(ring + stage * Shape::kStageBytes + b * Shape::kBox, cached ? paged : drafted, 64 * b,
                                p.kv_head, row, &full[stage]);
                ++put;
            };
            int id_before = -1, ids = -1; // tile j - 1's page; 32 tiles' pages
            for (int j = 0; j <= tiles; ++j)
            {
                int id = -1;
                if (Tree)
                {
                    if ((j & 31) == 0)
                    {
                        const int t = p.first_tile + j + lane;
                        ids = t < p.tiles_cached ? table[t] : -1;
                    }
                    id = __shfl_sync(0xFFFFFFFFu, ids, j & 31);
                }
                if (lane == 0)
                {
                    if (j < tiles)
                        load(j, &kmap, &kpages, id, keys, put_keys, KS, h.keys_full, h.keys_free);
                    if (j == 0 && ok && (i == 0 || one_wait(&h.query_free, (i - 1) & 1)))
                    {
                        mbar_expect_tx(&h.query, NQ * kBlocks * 128 * a.group * c.tile_tokens);
                        for (int b = 0; b < NQ * kBlocks; ++b)
                            tensor_load(queries + b * 128 * 128, &qmap, 64 * (b % kBlocks), p.kv_head * a.group,
                                        p.begin + p.token0 + b / kBlocks * c.tile_tokens, &h.query);
                        ++put_queries;
                    }
                    if (j > 0)
                        load(j - 1, &vmap, &vpages, id_before, values, put_values, VS, h.values_full, h.values_free);
                }
                id_before = id;
                __syncwarp();
            }
            ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
            leave(i);
        }
        // Every copy has landed before the CTA may end (only a failed run gets here early).
        if (lane == 0 && *(volatile int*) &h.dead)
        {
            if (put_queries)
                mbar_wait(&h.query, last_parity(put_queries));
            for (int n = max(0, put_keys - KS); n < put_keys; ++n)
                mbar_wait(&h.keys_full[n % KS], (n / KS) & 1);
            for (int n = max(0, put_values - VS); n < put_values; ++n)
                mbar_wait(&h.values_full[n % VS], (n / VS) & 1);
        }
        __syncwarp();
    }
    else if (warp == (NQ == 2 ? 13 : 3))
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
            const MmaPlace p = asked == 0 ? first : prompt_place(c, c.tile_tokens * NQ, unit);
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
    else if (warp <= NQ)
    {
        // S of query tile q.
        const int q = warp - 1;
        constexpr uint32_t kScores = tc_idesc16(kType, kKeyTile, false);
        const uint32_t qbase = smem_addr(queries) + q * Shape::kQueryBytes / NQ, kbase = smem_addr(keys);
        const uint32_t sbase = tmem + q * 2 * kKeyTile;
        int item = 0, count = 0; // key tiles, and those of q, before this
        bool ok = true;
        MmaPlace p;
        for (int i = 0; ok && take(i, p); ++i)
        {
            const int tiles = p.tiles, n = tiles_of(p, q);
            ok = wait(&h.query, i & 1);
            for (int j = 0; j < tiles && ok; ++j, ++item)
            {
                const int stage = item % KS;
                const bool reads = (lane & 1) && count > 0 && j < n; // S of the last tile is in registers
                ok = wait(reads ? &h.scores_read[q] : &h.keys_full[stage], (reads ? count - 1 : item / KS) & 1);
                if (!ok)
                    break;
                if (j < n)
                {
                    tc_fence_after();
#pragma unroll
                    for (int b = 0; b < D / 16; ++b)
                        tc_mma_warp(sbase, tc_desc(qbase + b / 4 * 128 * 128 + (b & 3) * 32),
                                    tc_desc(kbase + stage * Shape::kStageBytes + b / 4 * Shape::kBox + (b & 3) * 32), kScores,
                                    b > 0);
                    tc_commit_warp(&h.scores[q]);
                    ++count;
                }
                tc_commit_warp(&h.keys_free[stage]);
            }
            if (ok)
                tc_commit_warp(&h.query_free);
            leave(i);
        }
        finish_mmas(!*(volatile int*) &h.dead, &h.drained[q]);
    }
    else if (NQ == 2 ? warp == 3 || warp == 12 : warp == 2)
    {
        // O of query tile q.
        const int q = warp == 12 ? 1 : 0;
        constexpr uint32_t kRows = tc_idesc16(kType, D, true);
        const uint32_t vbase = smem_addr(values), wbase = tmem + q * 2 * kKeyTile + kKeyTile;
        const uint32_t obase = tmem + Shape::kScoreColumns + q * D;
        int item = 0, count = 0, rows = 0; // value tiles, those of q, and q's finished units before this
        bool ok = true;
        MmaPlace p;
        for (int i = 0; ok && take(i, p); ++i)
        {
            const int tiles = p.tiles, n = tiles_of(p, q);
            for (int j = 0; j < tiles && ok; ++j, ++item)
            {
                const int stage = item % VS;
                // The weights, and before a unit's first O the last one's in registers.
                const bool weighs = (lane & 1) && j < n, frees = (lane & 3) == 2 && j == 0 && j < n && rows > 0;
                ok = wait(frees ? &h.rows_free[q] : weighs ? &h.weights[q][count & 1] : &h.values_full[stage],
                          (frees ? rows - 1 : weighs ? count / 2 : item / VS) & 1);
                if (!ok)
                    break;
                if (j < n)
                {
                    const int t = p.first_tile + j;
                    const int valid = !Tree                 ? p.length - j * kKeyTile
                                      : t < p.tiles_cached ? p.cached - t * kKeyTile
                                                            : p.length;
                    if (valid < kKeyTile) // by each of the warps for its own MMAs
                    {
                        const int bytes = (kKeyTile - valid) * 128;
                        for (int b = 0; b < kBlocks; ++b)
                            for (int e = lane * 16; e < bytes; e += 512)
                                *reinterpret_cast<uint4*>(values + stage * Shape::kStageBytes + b * Shape::kBox + valid * 128
                                                          + e) = make_uint4(0, 0, 0, 0);
                        fence_proxy_async();
                        __syncwarp();
                    }
                    tc_fence_after();
#pragma unroll
                    for (int b = 0; b < kKeyTile / 16; ++b)
                        tc_mma_ts_warp(obase, wbase + (count & 1) * 32 + b * 8,
                                       tc_desc_mn(vbase + stage * Shape::kStageBytes + b * 2048, Shape::kBox), kRows,
                                       j > 0 || b > 0);
                    tc_commit_warp(&h.done[q][count & 1]);
                    ++count;
                }
                tc_commit_warp(&h.values_free[stage]);
            }
            rows += n > 0;
            leave(i);
        }
        finish_mmas(!*(volatile int*) &h.dead, &h.drained[2 + q]);
    }
    else if (warp >= 4 && warp < 4 + 4 * NQ)
    {
        const int q = (warp - 4) >> 2, quarter = warp & 3;
        const int row = quarter * 32 + lane; // the TMEM lane
        const uint32_t lanes = tmem + ((uint32_t) (quarter * 32) << 16);
        const uint32_t obase = lanes + Shape::kScoreColumns + q * D, sbase = lanes + q * 2 * kKeyTile;
        const float scale = a.scale_log2;
        int count = 0; // tiles before this
        bool ok = true;
        MmaPlace p;
        for (int i = 0;; ++i)
        {
            const bool stop = !ok || !take(i, p);
            if (Tree ? any_stops(1 + q, 128, stop) : stop)
                break;
            const int n = tiles_of(p, q);
            const int token = p.token0 + q * c.tile_tokens + row / a.group, head = p.kv_head * a.group + row % a.group;
            const bool real = row < c.tile_tokens * a.group && token < p.length;
            const bool idle = !__any_sync(0xFFFFFFFFu, real); // no row of the warp's: it keeps the others' step only
            const int* table = Tree ? a.table + (size_t) p.sequence * a.table_stride : nullptr;
            unsigned long long path = 0;
            if (Tree)
            {
                // The sequence's parents, and a row's path from them.
                int* parents = h.parents[i & 1];
                for (int e = tid & 127; e < p.length; e += 128)
                    parents[e] = a.parents[p.begin + e];
                named_sync(1 + q, 128);
                if (real)
                    path = tree_path(parents, token);
            }
            float m = -INFINITY, l = 0.f;
            int id = Tree && p.first_tile < p.tiles_cached ? table[p.first_tile] : -1;
            for (int j = 0; j < n; ++j, ++count)
            {
                const int t = p.first_tile + j;
                const int id_next = Tree && t + 1 < p.tiles_cached ? table[t + 1] : -1;
                // S is there, and the weights' buffer has been read (two tiles back).
                const bool frees = (lane & 1) && count >= 2;
                ok = wait(frees ? &h.done[q][count & 1] : &h.scores[q], (frees ? count / 2 - 1 : count) & 1);
                if (!ok)
                    break;
                tc_fence_after();
                if (idle)
                {
                    if (lane == 0)
                    {
                        mbar_arrive(&h.scores_read[q]);
                        mbar_arrive(&h.weights[q][count & 1]);
                    }
                    continue;
                }
                uint32_t r[64];
                tc_ld32(sbase, r);
                tc_ld32(sbase + 32, r + 32);
                tc_wait_ld32(r);
                tc_wait_ld32(r + 32);
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&h.scores_read[q]);
                float* s = reinterpret_cast<float*>(r);
                // What the row does not attend to.
                bool masked = true;
                if (Tree && t >= p.tiles_cached)
                {
#pragma unroll
                    for (int e = 0; e < 64; ++e)
                        s[e] = path >> e & 1 ? s[e] : -INFINITY;
                }
                else
                {
                    const int limit = !Tree                        ? token - j * kKeyTile + 1
                                      : page_there(id, a.pages) ? p.cached - t * kKeyTile
                                                                 : 0;
                    masked = __any_sync(0xFFFFFFFFu, limit < kKeyTile);
                    if (masked)
                    {
#pragma unroll
                        for (int e = 0; e < 64; ++e)
                            s[e] = e < limit ? s[e] : -INFINITY;
                    }
                }
                id = id_next;
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int e = 4; e < 60; e += 8)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        top[g] = max3_nan(top[g], s[e + 2 * g], s[e + 2 * g + 1]);
                const float m_tile = max3_nan(max3_nan(top[0], s[60], s[61]), max3_nan(top[1], s[62], s[63]),
                                              max_nan(top[2], top[3]))
                                     * scale;
                // A score of NaN or infinity, of which exp2_poly would make a number: the row is taken again.
                if (!(m_tile < INFINITY))
                    l = NAN;
                if (j == 0)
                    m = m_tile;
                else
                {
                    const bool rises = m_tile > m + 8.f;
                    if (__any_sync(0xFFFFFFFFu, rises))
                    {
                        // O of the last tile is complete before it is scaled.
                        ok = wait(&h.done[q][(count - 1) & 1], ((count - 1) / 2) & 1);
                        if (!ok)
                            break;
                        tc_fence_after();
                        const float alpha = rises ? exp2_approx(m - m_tile) : 1.f;
                        l *= alpha;
                        m = rises ? m_tile : m;
#pragma unroll 1
                        for (int b = 0; b < D; b += 16)
                        {
                            uint32_t o[16];
                            tc_ld16(obase + b, o);
                            tc_wait_ld(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                            tc_st16(obase + b, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : -m;
                uint32_t w[32];
                l += masked ? weigh<T, false>(s, scale, base, w) : weigh<T, true>(s, scale, base, w);
                tc_st32(sbase + kKeyTile + (count & 1) * 32, w);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&h.weights[q][count & 1]);
            }
            if (n > 0)
            {
                ok = ok && wait(&h.done[q][(count - 1) & 1], ((count - 1) / 2) & 1);
                tc_fence_after();
                const int at = p.begin + token; // the row of q and out
                const size_t part = (size_t) p.part * c.part_rows + row;
                const bool whole = !Tree || p.whole;
                // Nothing attended: 0 (O is 0, or NaN and the row taken again).
                const float scaled = !ok ? NAN : l == 0.f ? 0.f : whole ? 1.f / l : 1.f;
                // Stays 0 for finite values. A maximum of minus infinity may be of masked keys or
                // of such scores.
                float2 check = make_float2(l * 0.f, m == -INFINITY ? NAN : 0.f);
                char* mine = whole ? (char*) ((T*) a.out + at * a.out_stride + (size_t) head * a.width)
                                   : (char*) (c.part_o + part * a.width);
                const unsigned rows = __ballot_sync(0xFFFFFFFFu, real);
                char* four[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    four[k] = (char*) __shfl_sync(0xFFFFFFFFu, (unsigned long long) mine, (lane & ~3) + k);
#pragma unroll 1
                for (int b = 0; b < a.width && !idle; b += 32)
                {
                    uint32_t o[32];
                    tc_ld32(obase + b, o);
                    tc_wait_ld32(o);
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
                    {
                        const float2 v = make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1]));
                        check = __ffma2_rn(v, make_float2(0.f, 0.f), check);
                        const float2 y = __fmul2_rn(v, make_float2(scaled, scaled));
                        o[e] = __float_as_uint(y.x);
                        o[e + 1] = __float_as_uint(y.y);
                    }
                    uint32_t x[16];
                    if (whole)
                    {
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            x[e] = pack_pair<T>(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
                        store_rows(x, four, rows, 2 * b, 2 * a.width);
                    }
                    else
                    {
#pragma unroll
                        for (int g = 0; g < 2; ++g)
                        {
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                x[e] = o[16 * g + e];
                            store_rows(x, four, rows, 4 * (b + 16 * g), 4 * a.width);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&h.rows_free[q]);
                if (Tree && !whole && real)
                    c.part_ml[part] = make_float2(m, l);
                if (Tree && real && p.first_tile == 0 && row % a.group == 0)
                    c.spans[(size_t) at * a.kv_heads + p.kv_head] = span_of(p, blockIdx.x);
                // Rows that came out not finite: again, from what they attend to only.
                unsigned again = __ballot_sync(0xFFFFFFFFu, ok && real && !(check.x + check.y == 0.f));
                while (again)
                {
                    const int who = __ffs(again) - 1;
                    again &= again - 1;
                    const int at1 = __shfl_sync(0xFFFFFFFFu, at, who), head1 = __shfl_sync(0xFFFFFFFFu, head, who);
                    take_again<T, Tree>(c, h.place[i & 1], at1, head1);
                }
            }
            leave(i);
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 1)
        tc_dealloc(tmem, Shape::kTmem);
}

// Joins a query tile's parts: a warp a (row, head), lane c the channels [8 c, 8 c +
// 8). What one CTA held whole is finished already.
template <typename T>
__global__ void __launch_bounds__(256) attention_join(const __grid_constant__ MmaCall c)
{
    const AttnCall& a = c.a;
    const long long unit = (long long) blockIdx.x * 8 + (threadIdx.x >> 5);
    const int row = (int) (unit / a.heads), head = (int) (unit % a.heads), at = (threadIdx.x & 31) * 8;
    // The offsets too are behind the wait: the kernel ahead has waited for who wrote them, but nothing says
    // that its trigger hands that on. (The search ahead of the wait: 0.3 us of 14 less.)
    pdl_wait();
    if (row >= a.rows)
        return;
    const int2 words = c.spans[(size_t) row * a.kv_heads + head / a.group]; // on its way beside the search
    const unsigned failed = __ldcg(&g_operator_error);
    int begin;
    const int s = sequence_of_row(a, row, begin), node = row - begin;
    if (s < 0 || node >= a.max_nodes)
        return;
    const KeySpan span = key_span(words.x, words.y, c.ctas);
    const bool few = span.few;
    const int from = span.first, to = span.last;
    if (from == to && !failed)
        return;
    const int within = node % c.tile_tokens * a.group + head % a.group;
    auto part_of = [&](int cta) { return (size_t) (2 * cta + (!few && cta == from)) * c.part_rows + within; };
    // 32 parts at a time, a lane's maximum and sum each; four parts' rows in flight.
    float m = -INFINITY, l = 0.f, acc[8] = {};
    for (int base = from; base <= to; base += 32)
    {
        const int lane = threadIdx.x & 31, count = min(32, to + 1 - base);
        const float2 ml = lane < count ? c.part_ml[part_of(base + lane)] : make_float2(-INFINITY, 0.f);
        const float m_new = fmaxf(m, warp_max(ml.y == 0.f ? -INFINITY : ml.x));
        const float alpha = m == m_new ? 1.f : exp2f(m - m_new);
        // A part in which nothing was attended weighs nothing.
        const float weight = ml.y == 0.f ? 0.f : ml.x == m_new ? 1.f : exp2f(ml.x - m_new);
        l = l * alpha + warp_sum(weight * ml.y);
        m = m_new;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            acc[e] *= alpha;
        for (int i = 0; i < count; i += 4)
        {
            float x[4][8] = {};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < count && at < a.width)
                    load8(c.part_o + part_of(base + i + k) * a.width + at, x[k]);
#pragma unroll
            for (int k = 0; k < 4; ++k)
            {
                const float w = __shfl_sync(0xFFFFFFFFu, weight, (i + k) & 31);
                if (i + k < count && w != 0.f)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        acc[e] = fmaf(w, x[k][e], acc[e]);
            }
        }
    }
    // A wait has run out (here or, until hf_cuda_operators_sync has told it, in an earlier
    // call): rows, parts and spans may be missing, so every row is NaN.
    const float inv = failed || !span.there ? NAN : finish_factor(m, l);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        acc[e] *= inv; // 0 where nothing was attended
    if (at < a.width)
        store8((T*) a.out + row * a.out_stride + (size_t) head * a.width + at, acc);
}
} // namespace hfk
