// Prints the plan (acfun_amd/csrc/q8_plan.hpp) of each line of the input:
//   gemm M N K gated cus    -> the tile, or none
//   fc M N K gated          -> one | two, and /rows where one is taken on a captured stream
//   quant rows K trans      -> fits or not
//   sample rows cols cus    -> parts per threads
#include <cstdio>
#include <cstring>

#include "../../acfun_amd/csrc/q8_plan.hpp"

using namespace acfun;

int main() {
    static const char* const names[] = {"FEW16", "FEW32", "FEW64", "MANY128", "MANY256"};
    char what[8];
    int a, b, c, gated, cus;
    while (std::scanf("%7s %d %d %d", what, &a, &b, &c) == 4) {
        if (!std::strcmp(what, "gemm")) {
            if (std::scanf("%d %d", &gated, &cus) != 2) return 1;
            const Q8Kind k = q8_choose(a, b, c, gated, cus);
            const bool fits = q8_mm_fits(a, b, c, gated);
            std::puts(fits ? names[k] : "none");
            if (fits && !q8_mm_fits(a, b, c, k, gated)) return 2;
        } else if (!std::strcmp(what, "fc")) {
            if (std::scanf("%d", &gated) != 1) return 1;
            const bool fit = q8_rows_fit(a, b, c, gated);
            std::printf("%s%s\n", fit && q8_rows_one(a, c) ? "one" : "two",
                        fit && a <= kCapturedRows ? "/rows" : "");
        } else if (!std::strcmp(what, "sample")) {
            const SamplePlan p = sample_plan(a, b, c);
            std::printf("%d %d %d\n", p.parts, p.per, p.threads);
            if (p.parts < 1 || p.parts > kSampleParts || (long long)p.parts * p.per < b) return 3;
            if (p.parts > 1 && (p.per % 1024 || (long long)(p.parts - 1) * p.per >= b)) return 4;
        } else {
            std::puts(q8_quant_fits(a, c) && q8_dequant_fits(a, b) ? "fits" : "not");
        }
    }
}
