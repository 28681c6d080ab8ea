// Calls registered functions of tvm_ffi_adapter.cc (compiled with the headers of ffi_stub) and prints what reaches the entry points
// of the tensor level, which are defined here.
#include <tvm/ffi/function.h>

#include <cstdio>

extern "C" {
void* TVMFFIEnvGetStream(int32_t, int32_t) { return nullptr; }
const char* tvmkv_last_error(void) { return "refused"; }
int tvmkv_dl_move_kept_tokens(const DLTensor* pages, const DLTensor* key_weights, const DLTensor* page_indptr, const DLTensor* page_indices,
                              const DLTensor* weight_page_indices, const DLTensor* kept, void*) {
  for (const DLTensor* t : {pages, key_weights, page_indptr, page_indices, weight_page_indices, kept}) std::printf("%d ", t != nullptr ? t->ndim : -1);
  return 0;
}
}

int main(int argc, char** argv) {
  using namespace tvm::ffi;
  DLTensor tensors[8] = {};
  for (int i = 0; i < 8; ++i) tensors[i].ndim = i;  // what tells them apart
  std::vector<Any> args;
  for (int i = 2; i < argc; ++i) args.push_back(argv[i][0] == '-' ? Any{} : Any{Tensor(&tensors[argv[i][0] - '0'])});
  try {
    functions().at(argv[1])(args);
  } catch (const std::exception& e) {
    std::printf("%s", e.what());
    return 1;
  }
  return 0;
}
