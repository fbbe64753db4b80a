// Prints the plan (acfun_amd/csrc/mx_plan.hpp) of each line of the input:
//   gemm M N K cus          -> the kind, or none
//   fc M N K elem cus       -> rows16 | rows32 | rows64 (one launch), two, or two/rows.. (two, but the
//                              one on a captured stream)
//   quant rows K trans      -> fits or not
#include <cstdio>
#include <cstring>

#include "../../acfun_amd/csrc/mx_plan.hpp"

using namespace acfun;

int main() {
    static const char* const names[] = {"FEW16", "FEW32", "FEW64", "MANY128", "MANY256"};
    char what[8];
    int a, b, c, elem, cus;
    while (std::scanf("%7s %d %d %d", what, &a, &b, &c) == 4) {
        if (!std::strcmp(what, "gemm")) {
            if (std::scanf("%d", &cus) != 1) return 1;
            double us;
            const MmKind k = mm_choose(a, b, c, cus, us);
            std::puts(us < kNever ? names[k] : "none");
            if ((us < kNever) != mm_fits(a, b, c)) return 2;
        } else if (!std::strcmp(what, "fc")) {
            if (std::scanf("%d %d", &elem, &cus) != 2) return 1;
            const FcPlan p = fc_plan(a, b, c, (size_t)elem, cus);
            if (p.one) std::printf("rows%d\n", 16 * p.tn);
            else if (p.captured) std::printf("two/rows%d\n", 16 * p.tn);
            else std::puts("two");
        } else {
            std::puts(mx_quant_fits(a, b, c) ? "fits" : "not");
        }
    }
}
