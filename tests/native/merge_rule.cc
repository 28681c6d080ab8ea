// When the merge of a split launch's shares takes eight at once (runtime_support.h).
#include <cstdio>
#include <cstdlib>

#include "../../tvm_amd/csrc/runtime_support.h"

int main() {
  for (int64_t workgroups : {1, 100, 256, 257, 768, 769, 4000}) {
    for (int shares = 2; shares <= 64; ++shares) {
      const bool half = tvmkv::merge_shares_at_once(workgroups, shares, false, 256);
      const bool single = tvmkv::merge_shares_at_once(workgroups, shares, true, 256);
      // two shares of many rows are not read eight times
      if (shares == 2 && workgroups > 256 && (half || single)) return std::printf("two shares at once\n"), 1;
      if (half != (shares == 2 ? workgroups <= 256 : shares <= 8 || shares % 8 > 1 + shares / 16)) return std::printf("fp16 %d\n", shares), 1;
      if (single != (shares == 2 ? workgroups <= 256 : shares < 8 || workgroups <= 768)) return std::printf("float32 %d\n", shares), 1;
    }
  }
  std::printf("all checks passed\n");
  return 0;
}
