// mx_groups_check.cpp -- the constants by which the gradient products divide a CTA, and the choice of the 4-bit product's kernel.  Exit code
// 0 = all hold.
#include <cstdio>

#include "../../cntk_b200/csrc/qagg_mx_groups.h"

template <class G>
int check(bool dense, int ctas)
{
    // an mbarrier's count is 1 at least, used or not
    if (G::convArrivals < 1 || G::denseArrivals < 1 || G::takenArrivals < 1)
        return 1;
    // one arrival per warp: the four of an expanding group, all loaders, all result warps, of every CTA
    if (G::convArrivals != 4 * ctas || (dense && G::denseArrivals != 4 * G::load * ctas) || G::takenArrivals != 4 * G::result * ctas)
        return 2;
    // the registers handed out are no more than the launch has, and that no more than an SM's
    const int handed = 128 * (G::regsMisc + G::regsExpand * G::expand + G::regsResult * G::result + G::regsLoad * G::load);
    if (handed > G::regsLaunch * G::threads || G::regsLaunch * G::threads > 65536 || G::threads > 1024)
        return 3;
    if (G::threads != 128 * (1 + G::expand + G::result + G::load))
        return 4;
    // tensor memory: accumulators, then expanded steps of 32 columns
    if (G::accumulators * G::widest + 32 * G::slots > (int) qagg::TMEM_COLS || G::slots < G::expand)
        return 5;
    return 0;
}

int main()
{
    const int rc[4] = {check<qagg::GradGroups<false, false>>(false, 1), check<qagg::GradGroups<false, true>>(false, 2), check<qagg::GradGroups<true, false>>(true, 1),
                       check<qagg::GradGroups<true, true>>(true, 2)};
    for (int i = 0; i < 4; ++i)
        if (rc[i])
            return 10 * (i + 1) + rc[i];
    // where one kernel was measured to be clearly ahead, it is the one that is taken
    const struct
    {
        long long O, T, K;
        bool few;
    } measured[] = {{2048, 1, 2048, true}, {9304, 1, 2048, true}, {9304, 1, 4096, true}, {12288, 1, 4096, false}, {16384, 1, 4096, false}, {2048, 2, 2048, true},
                    {9304, 2, 2048, true}, {12288, 2, 2048, false}, {9304, 2, 4096, false}, {2048, 3, 2048, true}, {2048, 4, 2048, true}, {9304, 3, 512, false},
                    {9304, 4, 512, false}, {4096, 3, 2048, false}, {4096, 4, 2048, false}, {9304, 4, 1024, false}, {33, 4, 8192, true}};
    for (const auto& m : measured)
        if (qagg::times_few(m.O, m.T, m.K) != m.few)
            return 100;
    // x has to fit; nothing to multiply, or more tokens, is the tiles' business
    if (qagg::times_few(33, 4, 8193) || qagg::times_few(33, 3, 8193) || qagg::times_few(20, 1, 32769) || !qagg::times_few(20, 1, 32768) || qagg::times_few(20, 1, 0) ||
        qagg::times_few(20, 5, 32) || qagg::times_few(1LL << 29, 1, 32768))
        return 101;
    std::puts("groups ok");
    return 0;
}
