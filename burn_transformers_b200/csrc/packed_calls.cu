// Entry points that take their arguments as one record: the values in the order of the function's parameters, without gaps.  A caller
// that converts each of two dozen arguments by itself (ctypes) takes 2.4 us for it, for a record 0.6; what a decode step
// calls once a layer is offered this way too.
#include <cstring>
#include <tuple>

#include "api.h"
#include "common.cuh"

namespace {

template <typename T>
T next(const unsigned char*& at) {
  T value;
  std::memcpy(&value, at, sizeof value);
  at += sizeof value;
  return value;
}

template <typename... Args>
int call(int (*function)(Args...), const void* record, int bytes) {
  BT_CHECK(bytes == (int)(sizeof(Args) + ...), "a record of %d bytes for arguments of %d", bytes, (int)(sizeof(Args) + ...));
  const unsigned char* at = static_cast<const unsigned char*>(record);
  const std::tuple<Args...> args{next<Args>(at)...};      // (in braces: from left to right)
  return std::apply(function, args);
}

}  // namespace

extern "C" int bt_qk_norm_rotary_packed(const void* record, int bytes) { return call(bt_qk_norm_rotary, record, bytes); }
extern "C" int bt_cache4_append_packed(const void* record, int bytes) { return call(bt_cache4_append, record, bytes); }
extern "C" int bt_cache4_gather_packed(const void* record, int bytes) { return call(bt_cache4_gather, record, bytes); }
extern "C" int bt_cache4_attention_packed(const void* record, int bytes) { return call(bt_cache4_attention, record, bytes); }
extern "C" int bt_cache4_decode_packed(const void* record, int bytes) { return call(bt_cache4_decode, record, bytes); }
extern "C" int bt_cache4_prompt_packed(const void* record, int bytes) { return call(bt_cache4_prompt, record, bytes); }
