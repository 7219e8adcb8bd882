// attention_join over spans and parts that a failed call leaves: run by test_serving_failures.py.
#include "attention_mma.cuh"

#include <cmath>
#include <cstdio>
#include <vector>

using namespace hfk;

namespace
{
template <typename T>
T* upload(const std::vector<T>& v)
{
    T* p = nullptr;
    cudaMalloc(&p, v.size() * sizeof(T));
    cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice);
    return p;
}
} // namespace

int main()
{
    constexpr int kRows = 7, kHeads = 2, kWidth = 8, kCtas = 4, kPartRows = 2;
    // Two rows of one node each a sequence; one kv head of two query heads.
    std::vector<int> offsets(kRows + 1);
    for (int i = 0; i <= kRows; ++i)
        offsets[i] = i;
    // Never written (bytes of 255), past the last CTA, backwards, far past, negative; then one CTA's and two CTAs'.
    const std::vector<int2> spans = {{-1, -1}, {1, kCtas}, {3, 1}, {kFew | 2, 0x7FFFFFFF}, {-5, 2}, {2, 2}, {kFew | 1, 2}};
    // part p of kPartRows rows: value p + 1 with weight 1 (m = 0, l = 1).
    std::vector<float> part_o;
    for (int p = 0; p < 2 * kCtas; ++p)
        part_o.insert(part_o.end(), kPartRows * kWidth, p + 1.f);
    MmaCall c = {};
    c.a.offsets = upload(offsets);
    c.a.sequences = kRows;
    c.a.rows = kRows;
    c.a.heads = kHeads;
    c.a.kv_heads = 1;
    c.a.group = kHeads;
    c.a.width = kWidth;
    c.a.out_stride = kHeads * kWidth;
    c.a.max_nodes = 1;
    c.tile_tokens = 64;
    c.ctas = kCtas;
    c.part_rows = kPartRows;
    c.part_o = upload(part_o);
    c.part_ml = upload(std::vector<float2>(2 * kCtas * kPartRows, make_float2(0.f, 1.f)));
    c.spans = upload(spans);
    std::vector<float> out(kRows * kHeads * kWidth, 7.f);
    c.a.out = upload(out);
    int wrong = 0;
    for (unsigned failed = 0; failed < 2; ++failed)
    {
        cudaMemcpyToSymbol(g_operator_error, &failed, sizeof(failed));
        cudaMemcpy(c.a.out, std::vector<float>(out.size(), 7.f).data(), out.size() * 4, cudaMemcpyHostToDevice);
        attention_join<float><<<(kRows * kHeads + 7) / 8, 256>>>(c);
        cudaMemcpy(out.data(), c.a.out, out.size() * 4, cudaMemcpyDeviceToHost);
        for (size_t i = 0; i < out.size(); ++i)
        {
            const int row = (int) i / (kHeads * kWidth);
            // Row 5 lies with one CTA, which has finished it; row 6 with CTAs 1 and 2: parts 2 and 4, values 3 and 5.
            const float expected = failed || row < 5 ? NAN : row == 5 ? 7.f : 4.f;
            if (std::isnan(expected) ? !std::isnan(out[i]) : out[i] != expected)
                std::printf("failed %u, row %d: %g for %g\n", failed, row, out[i], expected), ++wrong;
        }
    }
    const cudaError_t e = cudaDeviceSynchronize();
    std::printf("%d wrong, %s\n", wrong, cudaGetErrorString(e));
    return wrong || e != cudaSuccess;
}
