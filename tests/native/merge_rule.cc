// When the merge of a split launch's shares takes eight at once (runtime_support.h).
#include <cstdio>
#include <cstdlib>

#include "../../tvm_amd/csrc/runtime_support.h"

int main() {
  for (int64_t workgroups : {1, 100, 256, 257, 4000}) {
    for (bool into : {false, true}) {
      for (int shares = 2; shares <= 64; ++shares) {
        const bool few = workgroups <= 256 && !into;
        const bool half = tvmkv::merge_shares_at_once(workgroups, shares, false, into, 256);
        const bool single = tvmkv::merge_shares_at_once(workgroups, shares, true, into, 256);
        // two shares are never read eight times, whole groups of eight in fp16 go through loops
        if (shares == 2 && (half || single)) return std::printf("two shares at once\n"), 1;
        if (shares >= 8 && half) return std::printf("%d fp16 shares at once\n", shares), 1;
        if (half != ((shares >= 5 && shares <= 7) || (few && shares >= 3 && shares <= 7))) return std::printf("fp16 %d\n", shares), 1;
        if (single != (shares >= 6 || (few && shares >= 3))) return std::printf("float32 %d\n", shares), 1;
      }
    }
  }
  std::printf("all checks passed\n");
  return 0;
}
