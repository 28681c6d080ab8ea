// What the registration source uses of tvm-ffi, as small as its test needs: values, functions by name, conversion of arguments.
#ifndef TESTS_NATIVE_FFI_STUB_FUNCTION_H_
#define TESTS_NATIVE_FFI_STUB_FUNCTION_H_

#include <cstdint>
#include <functional>
#include <map>
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <utility>
#include <variant>
#include <vector>

#include "../../../../../include/tvmkv_dlpack.h"

namespace tvm {
namespace ffi {

class Tensor {
 public:
  Tensor() = default;
  explicit Tensor(DLTensor* t) : t_(t) {}
  const DLTensor* operator->() const { return t_; }

 private:
  DLTensor* t_ = nullptr;
};

template <class T>
using Optional = std::optional<T>;

class Function;
using Value = std::variant<std::monostate, int64_t, double, Tensor>;  // monostate: None
struct Any {
  Value value;
  template <class T>
  T cast() const {
    if (const T* x = std::get_if<T>(&value)) return *x;
    throw std::runtime_error("type mismatch");
  }
  template <class T>
  std::optional<T> try_cast() const {
    const T* x = std::get_if<T>(&value);
    return x != nullptr ? std::optional<T>(*x) : std::nullopt;
  }
};
struct PackedArgs {
  const std::vector<Any>* args;
  int size() const { return static_cast<int>(args->size()); }
  const Any& operator[](int i) const { return (*args)[i]; }
};

template <class T>
struct Convert {
  static T from(const Any& x) { return x.cast<T>(); }
};
template <class T>
struct Convert<std::optional<T>> {
  static std::optional<T> from(const Any& x) {
    if (std::holds_alternative<std::monostate>(x.value)) return std::nullopt;
    return x.cast<T>();
  }
};

class Function {
 public:
  using Packed = std::function<void(const std::vector<Any>&)>;
  static Function FromPacked(std::function<void(PackedArgs, Any*)> f) {
    return Function([f](const std::vector<Any>& args) {
      Any result;
      f(PackedArgs{&args}, &result);
    });
  }
  template <class F>
  static Function FromTyped(F f) {
    return Typed(f, &F::operator());
  }
  template <class R, class... A>
  static Function FromTyped(R (*f)(A...)) {
    return Call<R, A...>(f, std::index_sequence_for<A...>());
  }
  Function() = default;
  void operator()(const std::vector<Any>& args) const { packed_(args); }

 private:
  explicit Function(Packed packed) : packed_(std::move(packed)) {}
  template <class F, class R, class... A>
  static Function Typed(F f, R (F::*)(A...) const) {
    return Call<R, A...>(f, std::index_sequence_for<A...>());
  }
  template <class R, class... A, class F, size_t... I>
  static Function Call(F f, std::index_sequence<I...>) {
    return Function([f](const std::vector<Any>& args) {
      if (args.size() != sizeof...(A)) throw std::runtime_error("wrong number of arguments");
      (void)f(Convert<std::decay_t<A>>::from(args[I])...);
    });
  }
  Packed packed_;
};

inline std::map<std::string, Function>& functions() {
  static std::map<std::string, Function> all;
  return all;
}

struct Raise {
  [[noreturn]] void operator&(const std::ostream& s) const { throw std::runtime_error(dynamic_cast<const std::ostringstream&>(s).str()); }
};

}  // namespace ffi
}  // namespace tvm

#define TVM_FFI_THROW(kind) ::tvm::ffi::Raise() & ::std::ostringstream()
#define TVM_FFI_ICHECK(x) \
  if (!(x)) TVM_FFI_THROW(InternalError)
#define TVM_FFI_ICHECK_EQ(a, b) TVM_FFI_ICHECK((a) == (b))
#define TVM_FFI_STATIC_INIT_BLOCK()                                      \
  static void register_all();                                            \
  static const int registered = (register_all(), 0);                     \
  static void register_all()

#endif  // TESTS_NATIVE_FFI_STUB_FUNCTION_H_
