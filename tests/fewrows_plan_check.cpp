// CPU check of when the few-rows kernel of the microscaled products is taken and how it is launched
// (int4linear_b200/csrc/fp4_fewrows_plan.cuh), built with the sanitizer of undefined behaviour: sizes up to the largest that the
// operators accept, every number of rows the rule lets through.  Each form of the launch has to be reached by some size.
// Prints "FEWROWS_OK <cases>".
#include <algorithm>
#include <cstdio>
#include <set>

#include "../int4linear_b200/csrc/fp4_fewrows_plan.cuh"

using namespace i4l;

static std::set<int> seen_cols, seen_stages, seen_split;

template <bool kBlock16, bool kGated>
static int check(int m, int n, int k)
{
    using G = FewRowsGeo<kBlock16, kGated>;
    const FewRowsPlan p = fewrows_plan<kBlock16, kGated>(m, n, k, 148);
    const int steps = (k + kFewRowsStepK - 1) / kFewRowsStepK;
    seen_cols.insert(p.cols);
    seen_stages.insert(p.stages);
    seen_split.insert(p.split);
    if (p.n_pad % 16 || p.n_pad < std::min(m, 128) || p.n_pad > 128) return 1;
    if (p.split < 1 || p.split > 8 || p.split > steps) return 2;                   // (every CTA has a step)
    if (p.stages < std::min(2, (steps + p.split - 1) / p.split) || p.stages > kFewRowsMaxStages) return 3;
    if (G::kW * p.n_pad + p.stages * G::kScaleCols > p.cols) return 4;             // accumulators and scales fit
    if (p.smem < 1024 + p.stages * p.stage_bytes) return 5;
    if (p.split > 1 && p.smem < 1024 + G::kW * p.n_pad * kFewRowsTile * 4) return 6;  // and the partial sums
    if ((p.smem + 1024) / kSharedPerCol < p.cols) return 7;                        // co-resident CTAs share the columns
    if (p.smem + 2048 > kSmShared / 2) return 8;                                   // two to an SM, a KB each for the rest
    if (static_cast<long long>(p.tiles) * p.split * p.groups > 0x7FFFFFFF) return 9;
    return 0;
}

int main()
{
    const int top = 1 << 26;
    const int ns[] = {1, 16, 127, 128, 129, 1000, 1024, 4096, 4736, 4737, 5000, 6000, 7000, 10000, 14336, 28672, 1 << 20, top - 1, top};
    const int ks[] = {32, 64, 256, 288, 512, 1024, 2048, 4096, 6144, 6176, 8192, 14336, 65536, top};
    int cases = 0;
    for (int n : ns)
        for (int k : ks) {
            for (int m : {1000, 4096, 1 << 20, top - 1, top})  // (many rows are refused without an overflow)
                for (bool gated : {false, true})
                    if (fewrows_preferred(m, n, k, gated, 148)) { std::printf("FAIL taken: %d x %d x %d\n", m, n, k); return 1; }
            for (int m = 1; m <= 300; ++m)
                for (int form = 0; form < 4; ++form) {
                    const bool gated = form & 1;
                    if (!fewrows_preferred(m, n, k, gated, 148)) continue;
                    const int rc = form == 0 ? check<false, false>(m, n, k) : form == 1 ? check<false, true>(m, n, k)
                                 : form == 2 ? check<true, false>(m, n, k) : check<true, true>(m, n, k);
                    if (rc) { std::printf("FAIL %d: %d x %d x %d, form %d\n", rc, m, n, k, form); return 1; }
                    ++cases;
                }
        }
    if (seen_cols != std::set<int>{128, 256} || seen_stages != std::set<int>{1, 2, 3} || seen_split.size() != 8) {
        std::printf("FAIL: forms that no size reaches, or others; columns:");
        for (int v : seen_cols) std::printf(" %d", v);
        std::printf("; stages:");
        for (int v : seen_stages) std::printf(" %d", v);
        std::printf("; CTAs to a tile:");
        for (int v : seen_split) std::printf(" %d", v);
        std::printf("\n");
        return 1;
    }
    std::printf("FEWROWS_OK %d\n", cases);
    return 0;
}
