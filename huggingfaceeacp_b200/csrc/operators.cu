// libhf_cuda.so: the serving operators on device pointers of include/hf_cuda.h
// (paged cache steps, packed prompt attention, tree attention). They hold no
// state: every check is made on the host before the first launch.
#include <hf_cuda.h>

#include "attention_few.cuh"
#include "attention_short.cuh"
#include "attention_limbs.cuh"
#include "attention_mma.cuh"
#include "attention_rows.cuh"
#include "launch.cuh"
#include "pages.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>

using namespace hfk;

static_assert(kPagePositions == HF_PAGE_ROWS && kTreeNodes == HF_TREE_NODES, "the header's sizes");

namespace
{
// A function of the driver's, looked up once; null when it is not there.
template <typename F>
F driver_call(std::atomic<F>& known, const char* name)
{
    if (F f = known.load(std::memory_order_relaxed))
        return f;
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion(name, &f, 12000, cudaEnableDefault, &found) != cudaSuccess
        || found != cudaDriverEntryPointSuccess)
        return nullptr;
    known.store((F) f, std::memory_order_relaxed);
    return (F) f;
}

// Whether the calling thread has a current context: one that has not used the device
// yet has none, and tensor maps cannot be encoded there.
bool has_context()
{
    using Current = CUresult (*)(CUcontext*);
    static std::atomic<Current> known {nullptr};
    const Current current = driver_call(known, "cuCtxGetCurrent");
    CUcontext context = nullptr;
    return current && current(&context) == CUDA_SUCCESS && context;
}

// Makes the device that holds `p` current, and the caller's again at the end.
class DeviceOf
{
public:
    explicit DeviceOf(const void* p)
    {
        int device = 0;
        if (!on_device(p, &device))
            return;
        if (cudaGetDevice(&before) != cudaSuccess
            || ((device != before || !has_context()) && cudaSetDevice(device) != cudaSuccess))
        {
            status = HF_E_CUDA;
            return;
        }
        changed = device != before;
        current = device;
        status = HF_OK;
    }
    ~DeviceOf()
    {
        if (changed)
            cudaSetDevice(before);
    }
    DeviceOf(const DeviceOf&) = delete;

    // The other buffers of the call: on the same device too.
    template <typename... P>
    bool holds(const P*... p) const
    {
        return (here(p) && ...);
    }

    int status = HF_E_INVALID;
    int current = 0;

private:
    // By the driver's call: about a third of the runtime's time, and a call asks for ten
    // pointers.
    static bool on_device(const void* p, int* device)
    {
        using Query = CUresult (*)(unsigned, CUpointer_attribute*, void**, CUdeviceptr);
        static std::atomic<Query> known {nullptr};
        const Query query = driver_call(known, "cuPointerGetAttributes");
        unsigned type = 0;
        int ordinal = -1;
        CUpointer_attribute which[2] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL};
        void* values[2] = {&type, &ordinal};
        if (!query || query(2, which, values, (CUdeviceptr) p) != CUDA_SUCCESS || type != CU_MEMORYTYPE_DEVICE || ordinal < 0)
            return false;
        *device = ordinal;
        return true;
    }
    bool here(const void* p) const
    {
        int device = 0;
        return !p || (on_device(p, &device) && device == current);
    }
    int before = 0;
    bool changed = false;
};

int size_of(int dtype)
{
    return dtype == HF_DTYPE_F32 ? 4 : dtype == HF_DTYPE_BF16 || dtype == HF_DTYPE_F16 ? 2 : 0;
}

bool aligned(const void* p)
{
    return p && (uintptr_t) p % 16 == 0;
}

// An int32 array; `optional` ones may be null.
bool words(const void* p, bool optional = false)
{
    return p ? (uintptr_t) p % 4 == 0 : optional;
}

// A row stride in elements: the width when 0; false when rows would overlap or
// are not 16-byte aligned.
bool row_stride(int64_t* stride, int64_t width, int size)
{
    if (*stride == 0)
        *stride = width;
    return *stride >= width && *stride <= (int64_t) 1 << 40 && *stride * size % 16 == 0;
}

int status_of(cudaError_t e)
{
    return e == cudaSuccess ? HF_OK : HF_E_CUDA;
}

// ---- the cache ---------------------------------------------------------------

// Sizes only; the layer stride is filled in.
int check_cache_sizes(const hf_page_cache* cache, hf_page_cache* c)
{
    if (!cache)
        return HF_E_INVALID;
    *c = *cache;
    const int size = size_of(c->dtype);
    if (!size || c->layers < 1 || c->pages < 1 || c->sequences < 1 || c->table_stride < 1
        || c->table_stride > (1 << 20) || c->pages >= (1 << 25))
        return HF_E_INVALID;
    if (c->kv_width < 8 || c->kv_width % 8 || c->kv_width > (1 << 20))
        return HF_E_SHAPE;
    const int64_t layer = (int64_t) c->pages * kPagePositions * c->kv_width;
    if (c->layer_stride == 0)
        c->layer_stride = layer;
    return c->layer_stride >= layer && c->layer_stride * size % 16 == 0 ? HF_OK : HF_E_INVALID;
}

int check_cache(const hf_page_cache* cache, hf_page_cache* c)
{
    if (const int rc = check_cache_sizes(cache, c))
        return rc;
    return aligned(c->keys) && aligned(c->values) && words(c->table) && words(c->lengths) && words(c->refs) ? HF_OK : HF_E_INVALID;
}

uint64_t book_bytes(const hf_page_cache& c)
{
    const uint64_t copies = std::max(c.sequences, c.pages);
    return 4 * (4 + 3 * copies + 2 * (uint64_t) c.sequences + 2 * (uint64_t) c.pages);
}

PageBook book_of(const hf_page_cache& c, void* workspace)
{
    PageBook b = {};
    const int size = size_of(c.dtype);
    b.keys = (char*) c.keys;
    b.values = (char*) c.values;
    b.layer_bytes = c.layer_stride * size;
    b.row_bytes = c.kv_width * size;
    b.layers = c.layers;
    b.pages = c.pages;
    b.sequences = c.sequences;
    b.table_stride = c.table_stride;
    b.table = c.table;
    b.lengths = c.lengths;
    b.refs = c.refs;
    b.copy_count = (int*) workspace;
    b.copies = (PageCopy*) (b.copy_count + 4);
    b.per_sequence = (int*) (b.copies + std::max(c.sequences, c.pages));
    b.free_ids = b.per_sequence + 2 * (size_t) c.sequences;
    b.renamed = b.free_ids + c.pages;
    return b;
}

// The bookkeeping kernel, `Book<true>` where the book fits shared memory.
template <typename Kernel, typename... Args>
cudaError_t launch_book(Kernel small, Kernel large, std::atomic<uint64_t>& ready, int device, cudaStream_t stream,
                        const PageBook& b, Args... args)
{
    const int64_t words = book_words(b.pages, b.sequences);
    if (words > kSmallBook)
        return launch(true, large, dim3(1), dim3(kBookThreads), 0, stream, b, args...);
    const uint64_t bit = 1ull << (device & 63); // devices whose kernel has its shared memory
    if (!(ready.load(std::memory_order_relaxed) & bit))
    {
        const cudaError_t e = cudaFuncSetAttribute(small, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * kSmallBook);
        if (e != cudaSuccess)
            return e;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    return launch(true, small, dim3(1), dim3(kBookThreads), (size_t) words * 4, stream, b, args...);
}

int copy_rows(const PageBook& b, int most, int device, cudaStream_t stream)
{
    const long long units = (long long) most * b.layers * 2 * ((kPagePositions * b.row_bytes + 32767) / 32768);
    const int grid = (int) std::min<long long>(std::max<long long>(units, 1), (long long) sm_count(device) * 8);
    return status_of(launch(true, pages_copy_rows, dim3(grid), dim3(256), 0, stream, b));
}

// ---- the attentions -----------------------------------------------------------

// Checks of what both attentions share; fills the kernels' call.
int check_attention(int dtype, int heads, int kv_heads, int width, int rows, float scale)
{
    if (!size_of(dtype) || heads < 1 || kv_heads < 1 || rows < 1 || !(scale > 0.f) || !std::isfinite(scale))
        return HF_E_INVALID;
    if (heads % kv_heads || heads / kv_heads > 128 || width < 8 || width % 8 || width > 256
        || (int64_t) heads * width > (1 << 24))
        return HF_E_SHAPE;
    return HF_OK;
}

template <typename Call>
int check_rows(const Call& call, int size, int heads, int kv_heads, int width, AttnCall* a)
{
    int64_t q = call.q_stride, k = call.k_stride, v = call.v_stride, o = call.out_stride;
    if (!aligned(call.q) || !aligned(call.k) || !aligned(call.v) || !aligned(call.out) || !words(call.offsets)
        || !row_stride(&q, (int64_t) heads * width, size) || !row_stride(&k, (int64_t) kv_heads * width, size)
        || !row_stride(&v, (int64_t) kv_heads * width, size) || !row_stride(&o, (int64_t) heads * width, size))
        return HF_E_INVALID;
    a->q = call.q;
    a->k = call.k;
    a->v = call.v;
    a->out = call.out;
    a->q_stride = q;
    a->k_stride = k;
    a->v_stride = v;
    a->out_stride = o;
    a->offsets = call.offsets;
    a->rows = call.rows;
    a->heads = heads;
    a->kv_heads = kv_heads;
    a->group = heads / kv_heads;
    a->width = width;
    a->scale_log2 = (float) (call.scale * 1.4426950408889634);
    return HF_OK;
}

// ---- tensor maps ---------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder()
{
    static std::atomic<EncodeTiled> known {nullptr};
    return driver_call(known, "cuTensorMapEncodeTiled");
}

// [rows][heads][width] elements, rows `stride` elements apart, in boxes of 128
// bytes of channels x box_heads x box_rows with the 128-byte swizzle, or of `plain`
// channels without one; zeros outside.
bool encode_rows(CUtensorMap* map, int dtype, const void* base, int width, int heads, int64_t rows, int64_t stride,
                 int box_heads, int box_rows, int plain = 0)
{
    const EncodeTiled encode = encoder();
    const int size = size_of(dtype);
    const CUtensorMapDataType type = dtype == HF_DTYPE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : dtype == HF_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                              : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t dims[3] = {(cuuint64_t) width, (cuuint64_t) heads, (cuuint64_t) rows};
    const cuuint64_t strides[2] = {(cuuint64_t) width * size, (cuuint64_t) stride * size};
    const cuuint32_t box[3] = {(cuuint32_t) (plain ? plain : 128 / size), (cuuint32_t) box_heads, (cuuint32_t) box_rows};
    const cuuint32_t ones[3] = {1, 1, 1};
    return encode
           && encode(map, type, 3, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     plain ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
                  == CUDA_SUCCESS;
}

// ---- attention_mma ---------------------------------------------------------------
constexpr int kSms = 148; // a B200's; the work is cut for it wherever the call is checked

// What it costs a unit of a tree's to begin and to end, in key tiles (it is counted in
// where the tiles are shared out): 48 decode steps of 50 to 2500 tokens, 32 heads on 8
// of 128, bf16: 75 us with 0, 60 with 2, 60 with 4, 61 with 6; 48 trees of 15 nodes over
// 50 to 1500, fp32: 218, 187, 171, 164, of 50 to 3000, 8 heads on one of 256: 107, 91,
// 82, 86; on plain FMAs, 64 steps of 200 to 2048: 52, 47, 50, 54.
constexpr int kStart = 4, kFewStart = 2;

// A tree's CTAs, one a place on the GPU, and the rows of a part that it leaves.
int tree_ctas(int dtype, int width)
{
    return kSms * (dtype != HF_DTYPE_F32 && width <= 128 ? 2 : 1);
}

int part_rows(int heads, int kv_heads, int max_nodes)
{
    const int group = heads / kv_heads;
    return std::min(128 / group, max_nodes) * group;
}

// Whether a call of at most `keys` keys a row goes to attention_short, which takes
// 3.5 us and 0.07 us a key on the GPU, and some 0.3 us for 1000 keys of all rows
// where they fill it. Bounds where the other kernels become as fast (us on the GPU,
// short and other; a launch less saves 1 to 3 us of the caller's on top):
//  trees, one row of 21, 101, 251 keys: fp32 5.2 and 12.0, 10.7 and 14.2, 21 and 15;
//  bf16 4.9 and 9.9, 10.9 and 11.8, 21 and 11.7. 16 rows of 31: bf16 7.3 and 10.8; a tree
//  of 8 nodes on 60: fp32 10.1 and 17, bf16 9.6 and 9.9; of 40: fp32 37 and 19, bf16 31 and
//  10; a prompt of 8, 32, 64 tokens, 8 heads of 256: fp32 4.0 and 21, 5.9 and 22, 13.1 and
//  21; bf16 3.8 and 7.9, 5.2 and 8.1, 9.1 and 7.9; 32 heads of 128, 32 tokens: fp32 12.6
//  and 18.5, bf16 10.3 and 6.7.
bool is_short(const AttnCall& a, int dtype, bool tree, int64_t keys)
{
    const int64_t most = dtype == HF_DTYPE_F32 ? 32768 : tree ? 24576 : 8192; // keys of all rows
    return keys <= 112 && (int64_t) a.rows * a.heads * keys <= most;
}

template <bool Tree>
int short_call(int dtype, const AttnCall& a, cudaStream_t stream)
{
    const dim3 grid((unsigned) (a.rows * a.heads)), block(32 * kShortWarps);
    return status_of(dtype == HF_DTYPE_F32    ? launch(true, attention_short<float, Tree>, grid, block, 0, stream, a)
                     : dtype == HF_DTYPE_BF16 ? launch(true, attention_short<__nv_bfloat16, Tree>, grid, block, 0, stream, a)
                                              : launch(true, attention_short<__half, Tree>, grid, block, 0, stream, a));
}

template <typename T, int D, int NQ, bool Tree>
int launch_mma(const CUtensorMap (&maps)[5], const MmaCall& c, int64_t ctas, int device, cudaStream_t stream)
{
    using Shape = MmaShape<D, NQ>;
    const auto kernel = attention_mma<T, D, NQ, Tree>;
    static std::atomic<uint64_t> ready {0}; // devices whose kernel has its shared memory
    const uint64_t bit = 1ull << (device & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit))
    {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem) != cudaSuccess)
            return HF_E_CUDA;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    return status_of(launch(true, kernel, dim3((unsigned) ctas), dim3(Shape::kThreads), Shape::kSmem, stream, maps[0],
                            maps[1], maps[2], maps[3], maps[4], c));
}

template <typename T>
int packed_mma(int dtype, const AttnCall& a, int device, cudaStream_t stream)
{
    MmaCall c = {};
    c.a = a;
    c.tile_tokens = 128 / a.group;
    // Two query tiles a CTA read the keys half as often (300 prompts of 100 to 400 tokens,
    // 32 heads on 8 of 128: 345 us, with one tile 390); with fewer of them than SMs
    // the rows are spread over twice the CTAs instead. Of prompts of less than three
    // tiles a second one is mostly empty, and what a unit costs to begin and to end
    // counts: two CTAs a SM of one tile each overlap it (4096 prompts of up to 16 tokens:
    // 357 us, with two tiles 644; 2048 of up to 64: 267 and 366; 1000 of 50 to 150: 441
    // and 439).
    const int64_t pairs = (int64_t) a.rows * a.heads / 256;
    const bool shorts = a.rows < 3LL * c.tile_tokens * a.sequences;
    const int nq = a.width <= 128 && pairs >= kSms && !shorts ? 2 : 1;
    const int64_t ctas = ((int64_t) a.rows / (c.tile_tokens * nq) + a.sequences) * a.kv_heads;
    CUtensorMap maps[5] = {};
    if (!encode_rows(&maps[0], dtype, a.q, a.width, a.heads, a.rows, a.q_stride, a.group, c.tile_tokens)
        || !encode_rows(&maps[1], dtype, a.k, a.width, a.kv_heads, a.rows, a.k_stride, 1, kKeyTile)
        || !encode_rows(&maps[2], dtype, a.v, a.width, a.kv_heads, a.rows, a.v_stride, 1, kKeyTile))
        return HF_E_CUDA;
    if (ctas > INT32_MAX)
        return HF_E_SHAPE;
    if (a.width > 128)
        return launch_mma<T, 256, 1, false>(maps, c, ctas, device, stream);
    if (a.width > 64)
        return nq == 2 ? launch_mma<T, 128, 2, false>(maps, c, ctas, device, stream)
                       : launch_mma<T, 128, 1, false>(maps, c, ctas, device, stream);
    return nq == 2 ? launch_mma<T, 64, 2, false>(maps, c, ctas, device, stream)
                   : launch_mma<T, 64, 1, false>(maps, c, ctas, device, stream);
}

void tree_call(MmaCall* c, int dtype, const AttnCall& a, void* workspace)
{
    c->a = a;
    c->tile_tokens = 128 / a.group;
    c->ctas = tree_ctas(dtype, a.width);
    c->start = kStart;
    c->part_rows = part_rows(a.heads, a.kv_heads, a.max_nodes);
    c->part_o = (float*) workspace;
    c->part_ml = (float2*) (c->part_o + (size_t) 2 * c->ctas * c->part_rows * a.width);
    c->spans = (int2*) (c->part_ml + (size_t) 2 * c->ctas * c->part_rows);
}

template <typename T>
int join(const MmaCall& c, cudaStream_t stream)
{
    const dim3 grid((unsigned) (((int64_t) c.a.rows * c.a.heads + 7) / 8));
    return status_of(launch(true, attention_join<T>, grid, dim3(256), 0, stream, c));
}

template <typename T>
int tree_mma(int dtype, const AttnCall& a, void* workspace, int device, cudaStream_t stream)
{
    MmaCall c = {};
    tree_call(&c, dtype, a, workspace);
    const int ctas = c.ctas;
    CUtensorMap maps[5] = {};
    const int64_t positions = (int64_t) a.pages * kPagePositions;
    if (!encode_rows(&maps[0], dtype, a.q, a.width, a.heads, a.rows, a.q_stride, a.group, c.tile_tokens)
        || !encode_rows(&maps[1], dtype, a.k, a.width, a.kv_heads, a.rows, a.k_stride, 1, kKeyTile)
        || !encode_rows(&maps[2], dtype, a.v, a.width, a.kv_heads, a.rows, a.v_stride, 1, kKeyTile)
        || !encode_rows(&maps[3], dtype, a.key_pages, a.width, a.kv_heads, positions, a.kv_heads * a.width, 1, kKeyTile)
        || !encode_rows(&maps[4], dtype, a.value_pages, a.width, a.kv_heads, positions, a.kv_heads * a.width, 1, kKeyTile))
        return HF_E_CUDA;
    const int rc = a.width > 128  ? launch_mma<T, 256, 1, true>(maps, c, ctas, device, stream)
                   : a.width > 64 ? launch_mma<T, 128, 1, true>(maps, c, ctas, device, stream)
                                  : launch_mma<T, 64, 1, true>(maps, c, ctas, device, stream);
    return rc ? rc : join<T>(c, stream);
}

// ---- attention_limbs (fp32) --------------------------------------------------------
// A prompt's workspace: the halves of K and V, then the tiles' factors.
int limb_tiles(int rows, int sequences)
{
    return rows / kKeyTile + sequences;
}

uint64_t limb_bytes(int rows, int sequences, int kv_heads, int width)
{
    return 8 * (uint64_t) rows * kv_heads * width + 8 * (uint64_t) kv_heads * limb_tiles(rows, sequences);
}

template <int D, bool Tree>
int launch_limbs(const CUtensorMap (&maps)[4], const LimbCall& l, int64_t ctas, int device, cudaStream_t stream)
{
    using Shape = LimbShape<D, Tree>;
    const auto kernel = attention_limbs<D, Tree>;
    static std::atomic<uint64_t> ready {0}; // devices whose kernel has its shared memory
    const uint64_t bit = 1ull << (device & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit))
    {
        // The warpgroups' register shares assume this count at launch.
        cudaFuncAttributes f;
        if (cudaFuncGetAttributes(&f, kernel) != cudaSuccess || f.numRegs != Shape::kLaunchRegisters
            || cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem) != cudaSuccess)
            return HF_E_CUDA;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    return status_of(launch(true, kernel, dim3((unsigned) ctas), dim3(Shape::kThreads), Shape::kSmem, stream, maps[0],
                            maps[1], maps[2], maps[3], l));
}

int packed_limbs(const AttnCall& a, void* workspace, int device, cudaStream_t stream)
{
    LimbCall l = {};
    l.c.a = a;
    l.c.tile_tokens = 128 / a.group;
    l.limbs = (__half*) workspace;
    l.tiles = limb_tiles(a.rows, a.sequences);
    const size_t limb = (size_t) a.rows * a.kv_heads * a.width;
    l.factors = (float*) (l.limbs + 4 * limb);
    const int64_t ctas = ((int64_t) a.rows / l.c.tile_tokens + a.sequences) * a.kv_heads;
    if (ctas > INT32_MAX || a.kv_heads > 65535)
        return HF_E_SHAPE;
    CUtensorMap maps[4] = {};
    const int limb_of[4] = {0, 2, 1, 3}; // K hi, V hi, K lo, V lo
    for (int i = 0; i < 4; ++i)
        if (!encode_rows(&maps[i], HF_DTYPE_F16, l.limbs + limb_of[i] * limb, a.width, a.kv_heads, a.rows,
                         (int64_t) a.kv_heads * a.width, 1, kKeyTile))
            return HF_E_CUDA;
    if (launch(true, split_tiles, dim3(l.tiles, a.kv_heads, 2), dim3(256), 0, stream, l) != cudaSuccess)
        return HF_E_CUDA;
    return a.width > 128  ? launch_limbs<256, false>(maps, l, ctas, device, stream)
           : a.width > 64 ? launch_limbs<128, false>(maps, l, ctas, device, stream)
                          : launch_limbs<64, false>(maps, l, ctas, device, stream);
}

template <int D>
int launch_few(const AttnCall& a, const MmaCall& c, int device, cudaStream_t stream)
{
    using Shape = FewShape<D>;
    CUtensorMap maps[4] = {};
    const int64_t positions = (int64_t) a.pages * kPagePositions, kvw = (int64_t) a.kv_heads * a.width;
    if (!encode_rows(&maps[0], HF_DTYPE_F32, a.k, a.width, a.kv_heads, a.rows, a.k_stride, 1, kFewKeys, D)
        || !encode_rows(&maps[1], HF_DTYPE_F32, a.v, a.width, a.kv_heads, a.rows, a.v_stride, 1, kFewKeys, D)
        || !encode_rows(&maps[2], HF_DTYPE_F32, a.key_pages, a.width, a.kv_heads, positions, kvw, 1, kFewKeys, D)
        || !encode_rows(&maps[3], HF_DTYPE_F32, a.value_pages, a.width, a.kv_heads, positions, kvw, 1, kFewKeys, D))
        return HF_E_CUDA;
    static std::atomic<uint64_t> ready {0}; // devices whose kernel has its shared memory
    const uint64_t bit = 1ull << (device & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit))
    {
        if (cudaFuncSetAttribute(attention_few<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem) != cudaSuccess)
            return HF_E_CUDA;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    return status_of(launch(true, attention_few<D>, dim3(c.ctas), dim3(Shape::kThreads), Shape::kSmem, stream, maps[0],
                            maps[1], maps[2], maps[3], c));
}

int tree_limbs(const AttnCall& a, void* workspace, int device, cudaStream_t stream)
{
    LimbCall l = {};
    MmaCall& c = l.c;
    tree_call(&c, HF_DTYPE_F32, a, workspace);
    // Up to eight rows a kv head the FMAs keep up with HBM, and nothing has to be
    // turned into halves.
    if (c.part_rows <= kFewRows)
    {
        c.start = kFewStart;
        const int rc = a.width > 128  ? launch_few<256>(a, c, device, stream)
                       : a.width > 64 ? launch_few<128>(a, c, device, stream)
                                      : launch_few<64>(a, c, device, stream);
        return rc ? rc : join<float>(c, stream);
    }
    const int ctas = c.ctas;
    CUtensorMap maps[4] = {};
    const int64_t positions = (int64_t) a.pages * kPagePositions, kvw = (int64_t) a.kv_heads * a.width;
    if (!encode_rows(&maps[0], HF_DTYPE_F32, a.k, a.width, a.kv_heads, a.rows, a.k_stride, 1, kKeyTile)
        || !encode_rows(&maps[1], HF_DTYPE_F32, a.v, a.width, a.kv_heads, a.rows, a.v_stride, 1, kKeyTile)
        || !encode_rows(&maps[2], HF_DTYPE_F32, a.key_pages, a.width, a.kv_heads, positions, kvw, 1, kKeyTile)
        || !encode_rows(&maps[3], HF_DTYPE_F32, a.value_pages, a.width, a.kv_heads, positions, kvw, 1, kKeyTile))
        return HF_E_CUDA;
    const int rc = a.width > 128  ? launch_limbs<256, true>(maps, l, ctas, device, stream)
                   : a.width > 64 ? launch_limbs<128, true>(maps, l, ctas, device, stream)
                                  : launch_limbs<64, true>(maps, l, ctas, device, stream);
    return rc ? rc : join<float>(c, stream);
}

int check_packed_sizes(const hf_attention_packed* call)
{
    if (!call || call->sequences < 1)
        return HF_E_INVALID;
    return check_attention(call->dtype, call->heads, call->kv_heads, call->head_width, call->rows, call->scale);
}

int check_tree_sizes(const hf_page_cache* cache, hf_page_cache* c, const hf_attention_tree* call)
{
    if (const int rc = check_cache_sizes(cache, c))
        return rc;
    if (!call || call->layer < 0 || call->layer >= c->layers || call->max_nodes < 1 || call->max_length < 0)
        return HF_E_INVALID;
    if (const int rc = check_attention(c->dtype, call->heads, call->kv_heads, call->head_width, call->rows, call->scale))
        return rc;
    if (call->max_nodes > HF_TREE_NODES || c->kv_width != call->kv_heads * call->head_width)
        return HF_E_SHAPE;
    // The kernels count key tiles in 32 bits.
    const int64_t tokens = 128 / (call->heads / call->kv_heads), row_tiles = (call->max_nodes + tokens - 1) / tokens;
    if ((call->max_length / kKeyTile + 2 + kStart) * row_tiles > (1 << 30) / ((int64_t) c->sequences * call->kv_heads))
        return HF_E_SHAPE;
    return HF_OK;
}

uint64_t packed_workspace(const hf_attention_packed& call)
{
    return call.dtype == HF_DTYPE_F32 ? limb_bytes(call.rows, call.sequences, call.kv_heads, call.head_width) : 0;
}

uint64_t tree_workspace(const hf_page_cache& c, const hf_attention_tree& call)
{
    return (uint64_t) 2 * tree_ctas(c.dtype, call.head_width) * part_rows(call.heads, call.kv_heads, call.max_nodes)
           * (4 * call.head_width + 8)
           + (uint64_t) 8 * call.rows * call.kv_heads;
}
} // namespace

extern "C" {
int hf_cuda_operators_sync(int device, void* stream)
{
    int before = 0;
    if (cudaGetDevice(&before) != cudaSuccess || cudaSetDevice(device) != cudaSuccess)
        return HF_E_CUDA;
    unsigned error = 0;
    cudaError_t e = cudaStreamSynchronize((cudaStream_t) stream);
    if (e == cudaSuccess)
        e = cudaMemcpyFromSymbol(&error, g_operator_error, sizeof(error));
    if (e == cudaSuccess && error)
    {
        const unsigned none = 0;
        e = cudaMemcpyToSymbol(g_operator_error, &none, sizeof(none));
    }
    cudaSetDevice(before);
    return e != cudaSuccess ? HF_E_CUDA : error ? HF_E_DEVICE : HF_OK;
}

int hf_cuda_pages_workspace(const hf_page_cache* cache, uint64_t* bytes)
{
    hf_page_cache c;
    if (!bytes)
        return HF_E_INVALID;
    *bytes = 0;
    if (const int rc = check_cache_sizes(cache, &c))
        return rc;
    *bytes = book_bytes(c);
    return HF_OK;
}

int hf_cuda_pages_update(const hf_page_cache* cache, const int32_t* release, int32_t releases, const int32_t* forks,
                         int32_t fork_count, const int32_t* grow, int32_t* result, void* workspace,
                         uint64_t workspace_bytes, void* stream)
{
    hf_page_cache c;
    if (const int rc = check_cache(cache, &c))
        return rc;
    if (releases < 0 || releases > c.sequences || fork_count < 0 || fork_count > c.sequences || !words(result)
        || !words(release, !releases) || !words(forks, !fork_count) || !words(grow, true) || !aligned(workspace))
        return HF_E_INVALID;
    if (workspace_bytes < book_bytes(c))
        return HF_E_CAPACITY;
    const DeviceOf on(c.keys);
    if (on.status)
        return on.status;
    if (!on.holds(c.values, c.table, c.lengths, c.refs, releases ? release : nullptr, fork_count ? forks : nullptr, grow,
                  result, workspace))
        return HF_E_INVALID;
    const PageBook b = book_of(c, workspace);
    cudaStream_t s = (cudaStream_t) stream;
    static std::atomic<uint64_t> ready {0};
    const cudaError_t e = launch_book(pages_update_book<true>, pages_update_book<false>, ready, on.current, s, b, release,
                                      (int) releases, forks, (int) fork_count, grow, result);
    if (e != cudaSuccess || !grow)
        return status_of(e);
    return copy_rows(b, c.sequences, on.current, s);
}

int hf_cuda_pages_compact(const hf_page_cache* cache, int32_t* live, void* workspace, uint64_t workspace_bytes,
                          void* stream)
{
    hf_page_cache c;
    if (const int rc = check_cache(cache, &c))
        return rc;
    if (!words(live) || !aligned(workspace))
        return HF_E_INVALID;
    if (workspace_bytes < book_bytes(c))
        return HF_E_CAPACITY;
    const DeviceOf on(c.keys);
    if (on.status)
        return on.status;
    if (!on.holds(c.values, c.table, c.lengths, c.refs, live, workspace))
        return HF_E_INVALID;
    const PageBook b = book_of(c, workspace);
    cudaStream_t s = (cudaStream_t) stream;
    static std::atomic<uint64_t> ready {0};
    const cudaError_t e =
        launch_book(pages_compact_book<true>, pages_compact_book<false>, ready, on.current, s, b, live);
    if (e != cudaSuccess)
        return HF_E_CUDA;
    return copy_rows(b, c.pages / 2 + 1, on.current, s);
}

int hf_cuda_pages_write(const hf_page_cache* cache, int32_t layer, const void* k, const void* v, int64_t k_stride,
                        int64_t v_stride, int32_t source_rows, const int32_t* offsets, const int32_t* index,
                        int32_t rows, void* stream)
{
    hf_page_cache c;
    if (const int rc = check_cache(cache, &c))
        return rc;
    const int size = size_of(c.dtype);
    if (layer < 0 || layer >= c.layers || rows < 0 || source_rows < 0 || !words(offsets) || !words(index, true) || !aligned(k) || !aligned(v)
        || !row_stride(&k_stride, c.kv_width, size) || !row_stride(&v_stride, c.kv_width, size))
        return HF_E_INVALID;
    if (rows == 0 || source_rows == 0)
        return HF_OK;
    const DeviceOf on(c.keys);
    if (on.status)
        return on.status;
    if (!on.holds(c.values, c.table, c.lengths, k, v, offsets, index))
        return HF_E_INVALID;
    PageWrite w = {};
    w.keys = (char*) c.keys + layer * c.layer_stride * size;
    w.values = (char*) c.values + layer * c.layer_stride * size;
    w.k = (const char*) k;
    w.v = (const char*) v;
    w.k_stride = k_stride * size;
    w.v_stride = v_stride * size;
    w.row_bytes = c.kv_width * size;
    w.pages = c.pages;
    w.sequences = c.sequences;
    w.table_stride = c.table_stride;
    w.table = c.table;
    w.lengths = c.lengths;
    w.offsets = offsets;
    w.index = index;
    w.rows = rows;
    w.source_rows = source_rows;
    return status_of(launch(true, pages_write_rows, dim3((unsigned) (rows + 7) / 8), dim3(256), 0, (cudaStream_t) stream, w));
}

int hf_cuda_attention_packed_workspace(const hf_attention_packed* call, uint64_t* bytes)
{
    if (!bytes)
        return HF_E_INVALID;
    *bytes = 0;
    if (const int rc = check_packed_sizes(call))
        return rc;
    *bytes = packed_workspace(*call);
    return HF_OK;
}

int hf_cuda_attention_packed(const hf_attention_packed* call, void* stream)
{
    if (const int rc = check_packed_sizes(call))
        return rc;
    AttnCall a = {};
    if (const int rc = check_rows(*call, size_of(call->dtype), call->heads, call->kv_heads, call->head_width, &a))
        return rc;
    a.sequences = call->sequences;
    const uint64_t bytes = packed_workspace(*call);
    if (bytes && !aligned(call->workspace))
        return HF_E_INVALID;
    if (call->workspace_bytes < bytes)
        return HF_E_CAPACITY;
    const DeviceOf on(a.q);
    if (on.status)
        return on.status;
    if (!on.holds(bytes ? call->workspace : nullptr, a.k, a.v, a.out, a.offsets))
        return HF_E_INVALID;
    cudaStream_t st = (cudaStream_t) stream;
    if (is_short(a, call->dtype, false, a.rows))
        return short_call<false>(call->dtype, a, st);
    if (call->dtype == HF_DTYPE_F32)
        return packed_limbs(a, call->workspace, on.current, st);
    return call->dtype == HF_DTYPE_BF16 ? packed_mma<__nv_bfloat16>(call->dtype, a, on.current, st)
                                        : packed_mma<__half>(call->dtype, a, on.current, st);
}

int hf_cuda_attention_tree_workspace(const hf_page_cache* cache, const hf_attention_tree* call, uint64_t* bytes)
{
    hf_page_cache c;
    if (!bytes)
        return HF_E_INVALID;
    *bytes = 0;
    if (const int rc = check_tree_sizes(cache, &c, call))
        return rc;
    *bytes = tree_workspace(c, *call);
    return HF_OK;
}

int hf_cuda_attention_tree(const hf_page_cache* cache, const hf_attention_tree* call, void* stream)
{
    hf_page_cache c;
    if (const int rc = check_tree_sizes(cache, &c, call))
        return rc;
    AttnCall a = {};
    const int size = size_of(c.dtype);
    if (const int rc = check_rows(*call, size, call->heads, call->kv_heads, call->head_width, &a))
        return rc;
    if (!aligned(c.keys) || !aligned(c.values) || !words(c.table) || !words(c.lengths) || !words(call->parents))
        return HF_E_INVALID;
    a.sequences = c.sequences;
    a.parents = call->parents;
    a.key_pages = (const char*) c.keys + call->layer * c.layer_stride * size;
    a.value_pages = (const char*) c.values + call->layer * c.layer_stride * size;
    a.table = c.table;
    a.lengths = c.lengths;
    a.pages = c.pages;
    a.table_stride = c.table_stride;
    a.max_nodes = call->max_nodes;
    a.max_length = std::min(call->max_length, c.table_stride * kPagePositions);
    const uint64_t bytes = tree_workspace(c, *call);
    if (!aligned(call->workspace))
        return HF_E_INVALID;
    if (call->workspace_bytes < bytes)
        return HF_E_CAPACITY;
    const DeviceOf on(a.q);
    if (on.status)
        return on.status;
    if (!on.holds(call->workspace, a.k, a.v, a.out, a.offsets, a.parents, a.key_pages, a.value_pages, a.table, a.lengths))
        return HF_E_INVALID;
    cudaStream_t st = (cudaStream_t) stream;
    if (is_short(a, c.dtype, true, (int64_t) a.max_length + a.max_nodes))
        return short_call<true>(c.dtype, a, st);
    if (c.dtype == HF_DTYPE_F32)
        return tree_limbs(a, call->workspace, on.current, st);
    return c.dtype == HF_DTYPE_BF16 ? tree_mma<__nv_bfloat16>(c.dtype, a, call->workspace, on.current, st)
                                    : tree_mma<__half>(c.dtype, a, call->workspace, on.current, st);
}
}
