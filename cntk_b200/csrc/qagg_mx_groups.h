// qagg_mx_groups.h -- how the gradient products (qagg_mx_gemm.cu) divide a CTA's warps, registers and tensor memory, and which kernel a 4-bit
// product takes.  Nothing here needs a device compiler, so that a host compiler can check it.
#pragma once

namespace qagg {

constexpr unsigned TMEM_COLS = 512; // accumulators first; behind them block scales or expanded operands

// Threads, in groups of four warps: copy / product / allocating / spare; expanding; result; with a dense operand that the copy engine
// cannot take, fewer of the second and third kind and four groups of loaders.  The threads are launched with as many registers
// each as the SM has for all of them, and redistribute them.
// PAIR: two CTAs make a 256 x 256 tile together, each with 128 rows of the packed operand and half of dy's columns, so that each brings
// 24 KB (int8; fp4 20) for 512 cycles of products where a CTA by itself brings 32 (28) for 384: copies from L2, at some 46
// bytes a cycle, are what bounds these kernels.  With loaders the tile is 256 x 128, and each CTA splits 64 of the columns.
// Tensor memory: two accumulators of 192 columns and four expanded steps of 32, or, tiles being 128 wide with loaders, two of 128
// and eight.  A 192-wide tile reads 6 % more per product than one of 256, which would leave room for one accumulator.  A pair has one
// of 256 columns, and eight expanded steps.
constexpr int GRAD_WIDEST = 192, GRAD_WIDEST_DENSE = 128, GRAD_PAIR = 256;
template <bool DENSE, bool PAIR>
struct GradGroups
{
    static constexpr int expand = DENSE ? (PAIR ? 2 : 1) : PAIR ? 2 : 3, result = DENSE ? 1 : 2, load = DENSE ? 4 : 0;
    static constexpr int firstExpand = 4, firstResult = firstExpand + 4 * expand, firstLoad = firstResult + 4 * result;
    static constexpr int threads = 128 * (1 + expand + result + load);
    static constexpr int regsLaunch = DENSE ? (PAIR ? 64 : 72) : PAIR ? 96 : 80; // 65536 / threads, a multiple of 8
    static constexpr int regsMisc = DENSE ? 40 : PAIR ? 48 : 56, regsExpand = DENSE && PAIR ? 48 : PAIR ? 64 : 56, regsResult = DENSE || PAIR ? 152 : 128,
                         regsLoad = PAIR ? 56 : 64;
    static_assert(regsLaunch * threads <= 65536 && 128 * (regsMisc + regsExpand * expand + regsResult * result + regsLoad * load) <= regsLaunch * threads, "registers");
    static constexpr int widest = DENSE ? GRAD_WIDEST_DENSE : PAIR ? GRAD_PAIR : GRAD_WIDEST;
    static constexpr int accumulators = PAIR && !DENSE ? 1 : 2;
    static constexpr unsigned side = accumulators * widest;     // first column behind the accumulators
    static constexpr int slots = (int) (TMEM_COLS - side) / 32; // expanded steps in tensor memory
    // Warps that arrive at a barrier in each phase: four of the group that has a step expanded it, all loaders wrote their part, all result
    // warps took the accumulator; a pair's arrive at the first CTA's barriers.  A barrier takes a count of 1 at least, and the dense one is
    // set up without loaders too.
    static constexpr int convArrivals = PAIR ? 8 : 4, denseArrivals = DENSE ? 4 * load * (PAIR ? 2 : 1) : 1, takenArrivals = 4 * result * (PAIR ? 2 : 1);
    static_assert(convArrivals >= 1 && denseArrivals >= 1 && takenArrivals >= 1, "barrier counts");
};

// A 4-bit product y (O x T) of K inputs: by the kernel for a few tokens, or by tiles on the tensor cores?  The few tokens' x, a byte a value,
// stays in shared memory.  Two tokens at most: until the integer dot products last longer than what the tiles need besides the weights.
// Three and four (both computed as four) bring twice the work for the same weights, and cross the tiles earlier.
// us, this / tiles, weights in L2:  1 token 2048 x 2048 2.4 / 4.8, 9304 x 2048 4.5 / 6.2, 9304 x 4096 6.8 / 7.1, 9304 x 4608 8.0 / 7.7;
// 2 tokens 9304 x 2048 5.5 / 6.3, 4096 x 4096 6.0 / 5.9, 12288 x 2048 7.4 / 6.3;  4 tokens 2048 x 2048 4.0 / 5.0, 9304 x 512 5.7 / 4.1,
// 2048 x 4096 5.9 / 5.8, 4096 x 2048 5.7 / 5.1.  With the weights in HBM both take half a microsecond to a whole one more.
constexpr long long FEW = 4, FEW_VALUES = 32768;
constexpr bool times_few(long long O, long long T, long long K)
{
    const long long t = T == 3 ? 4 : T;
    return T >= 1 && T <= FEW && K > 0 && t * K <= FEW_VALUES && t * O * K <= (T <= 2 ? 38LL << 20 : 16LL << 20);
}

} // namespace qagg
