// How a block's warps trade registers (setmaxnreg), and what has to hold for it. Plain C++.
#pragma once

namespace mxb200 {

// The first `few_warps` warps go down to `few` registers a thread, the other `many_warps` up to `many`. What the latter draw is
// what the block was launched with, its threads times the registers that the compiler gave the kernel, and not what else the SM
// has: where that is too little, setmaxnreg.inc waits for ever, and no bounded wait of the kernel ends it. The compiler's number
// may differ from build to build, so every launch of such a kernel is preceded by a look at it.
struct RegisterSplit {
  int few_warps = 0, few = 0, many_warps = 0, many = 0;

  // per thread, as launched; 0: nothing is traded
  constexpr int needed() const {
    const int warps = few_warps + many_warps;
    return warps == 0 ? 0 : (few_warps * few + many_warps * many + warps - 1) / warps;
  }
  // Whether a kernel that the compiler gave `registers` a thread may run: neither waits nor goes "down" to more than it has.
  constexpr bool served_by(int registers) const { return registers >= needed() && (few_warps == 0 || registers >= few); }
};

}  // namespace mxb200
