// Entry points by number, their arguments in 8-byte slots: a caller whose foreign
// function interface pays per argument (40 of them: 3.8 us from Python) packs
// them in one step and passes two (1.1 us).
#include <cstring>
#include <limits>
#include <tuple>
#include <type_traits>
#include <utility>

#include "common.cuh"

namespace mz {
namespace {

// Slot `i` as a T; *ok stays true where its value is one of T's.
template <class T>
T slot(const unsigned char *slots, size_t i, bool *ok) {
  if constexpr (std::is_floating_point<T>::value) {
    double x;
    memcpy(&x, slots + 8 * i, 8);
    return static_cast<T>(x);
  } else if constexpr (std::is_pointer<T>::value) {
    uint64_t x;
    memcpy(&x, slots + 8 * i, 8);
    return reinterpret_cast<T>(static_cast<uintptr_t>(x));
  } else {
    int64_t x;
    memcpy(&x, slots + 8 * i, 8);
    if (sizeof(T) < 8 && (x < static_cast<int64_t>(std::numeric_limits<T>::min()) ||
                          x > static_cast<int64_t>(std::numeric_limits<T>::max())))
      *ok = false;
    return static_cast<T>(x);
  }
}

template <class... A, size_t... I>
int unpack(int (*f)(A...), const unsigned char *slots, const char *name,
           std::index_sequence<I...>) {
  bool ok = true;
  const std::tuple<A...> args{slot<A>(slots, I, &ok)...};
  if (!ok) return fail(MZ_ERR_INVALID_ARG, "%s: an argument is out of its type's range", name);
  return f(std::get<I>(args)...);
}

template <class... A>
int call(int (*f)(A...), const void *slots, int n_slots, const char *name) {
  if (!slots || n_slots != static_cast<int>(sizeof...(A)))
    return fail(MZ_ERR_INVALID_ARG, "%s: takes %d arguments", name, static_cast<int>(sizeof...(A)));
  return unpack(f, static_cast<const unsigned char *>(slots), name, std::index_sequence_for<A...>());
}

}  // namespace
}  // namespace mz

extern "C" int mz_call_packed(int32_t op, const void *slots, int32_t n_slots) {
#define MZ_PACKED(op_, f_) \
  case op_: return mz::call(f_, slots, n_slots, #f_)
  switch (op) {
    MZ_PACKED(MZ_OP_PAGED_PLAN, mz_paged_plan);
    MZ_PACKED(MZ_OP_QK_NORM_ROPE, mz_qk_norm_rope);
    MZ_PACKED(MZ_OP_PAGED_DECODE_MOD, mz_paged_decode_mod);
    MZ_PACKED(MZ_OP_PAGED_APPEND_DECODE_MOD, mz_paged_append_decode_mod);
    MZ_PACKED(MZ_OP_PAGED_PREFILL_MOD, mz_paged_prefill_mod);
  }
#undef MZ_PACKED
  return mz::fail(MZ_ERR_INVALID_ARG, "mz_call_packed: no entry point %d", op);
}
