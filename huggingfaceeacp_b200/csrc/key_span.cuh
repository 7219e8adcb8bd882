// Which CTAs of a tree call hold a row's keys, as the CTA that begins the row's query
// tile leaves it for attention_join. Plain C++, so that it is tested without a GPU.
#pragma once

#ifdef __CUDACC__
#define HFK_BOTH __host__ __device__
#else
#define HFK_BOTH
#endif

namespace hfk
{
constexpr int kFew = 1 << 30; // in the first CTA's word: the row of tiles was cut for few query tiles

struct KeySpan
{
    int first, last;
    bool few;
    bool there; // a span that a CTA of the call can have left
};

// A call in which a wait ran out leaves spans unwritten: what the workspace holds
// there may be anything, and becomes a span of no CTA.
HFK_BOTH inline KeySpan key_span(int x, int y, int ctas)
{
    const int first = x & ~kFew;
    if (first < 0 || first > y || y >= ctas)
        return {0, -1, false, false};
    return {first, y, (x & kFew) != 0, true};
}
} // namespace hfk
