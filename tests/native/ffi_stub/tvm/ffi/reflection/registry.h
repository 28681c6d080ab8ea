#pragma once
#include "../function.h"
namespace tvm {
namespace ffi {
namespace reflection {
struct GlobalDef {
  template <class F>
  GlobalDef& def(const char* name, F f) {
    functions()[name] = Function::FromTyped(f);
    return *this;
  }
  template <class F>
  GlobalDef& def_packed(const char* name, F f) {
    functions()[name] = Function::FromPacked(f);
    return *this;
  }
};
}  // namespace reflection
}  // namespace ffi
}  // namespace tvm
