// The serving operators' entry point for arguments in a record.
#include <cuda_runtime.h>

#include <climits>
#include <cstdio>
#include <cstring>

#include "../../include/frcuda.h"
#include "kv_q4.cuh"

namespace {

// Eight-byte words; an integer that its parameter cannot hold becomes INT_MIN,
// which no operator takes.
struct Record {
  const unsigned char* at;
  template <typename T>
  T word(int i) const {
    T v;
    std::memcpy(&v, at + 8 * i, 8);
    return v;
  }
  int64_t i64(int i) const { return word<int64_t>(i); }
  int i32(int i) const {
    const int64_t v = i64(i);
    return v < INT_MIN || v > INT_MAX ? INT_MIN : static_cast<int>(v);
  }
  float real(int i) const { return static_cast<float>(word<double>(i)); }
  template <typename T>
  T* ptr(int i) const {
    return word<T*>(i);
  }
};

}  // namespace

extern "C" int frc_serving_call(int op, const void* record, size_t bytes, void* stream) {
  FRC_REQUIRE(record, "frc_serving_call: null pointer");
  const Record a{static_cast<const unsigned char*>(record)};
  switch (op) {
    case FRC_OP_QK_NORM_ROPE:
      FRC_REQUIRE(bytes == 24 * 8, "frc_serving_call: the record has another size");
      return frc_qk_norm_rope(a.i32(0), a.i32(1), a.ptr<const void>(2), a.i64(3), a.i64(4), a.i32(5), a.i32(6),
                              a.i32(7), a.ptr<const float>(8), a.ptr<const float>(9), a.ptr<const float>(10),
                              a.real(11), a.ptr<const float>(12), a.ptr<const float>(13), a.i64(14), a.i32(15),
                              a.i32(16), a.ptr<const int>(17), a.ptr<void>(18), a.i64(19), a.ptr<void>(20),
                              a.i64(21), a.ptr<void>(22), a.i64(23), stream);
    case FRC_OP_KV_APPEND_Q4:
      FRC_REQUIRE(bytes == 14 * 8, "frc_serving_call: the record has another size");
      return frc_kv_append_q4(a.i32(0), a.ptr<const void>(1), a.i64(2), a.i64(3), a.ptr<const void>(4), a.i64(5),
                              a.i64(6), a.i64(7), a.ptr<const int64_t>(8), a.i32(9), a.i32(10), a.i64(11),
                              a.i32(12), a.ptr<void>(13), stream);
    case FRC_OP_KV_READ_Q4:
      FRC_REQUIRE(bytes == 14 * 8, "frc_serving_call: the record has another size");
      return frc_kv_read_q4(a.i32(0), a.ptr<const void>(1), a.ptr<const int64_t>(2), a.i64(3), a.i32(4), a.i32(5),
                            a.i64(6), a.i32(7), a.ptr<void>(8), a.i64(9), a.i64(10), a.ptr<void>(11), a.i64(12),
                            a.i64(13), stream);
    case FRC_OP_ATTENTION_DECODE_Q4:
      FRC_REQUIRE(bytes == 21 * 8, "frc_serving_call: the record has another size");
      return frc_attention_decode_q4(a.i32(0), a.ptr<const void>(1), a.i64(2), a.i64(3), a.ptr<const void>(4),
                                     a.i64(5), a.i32(6), a.ptr<const int>(7), a.i64(8), a.i32(9),
                                     a.ptr<const int>(10), a.i32(11), a.i32(12), a.i32(13), a.i32(14), a.real(15),
                                     a.ptr<void>(16), static_cast<size_t>(a.i64(17)), a.ptr<void>(18), a.i64(19),
                                     a.i64(20), stream);
    case FRC_OP_ATTENTION_PREFILL:
      FRC_REQUIRE(bytes == 23 * 8, "frc_serving_call: the record has another size");
      return frc_attention_prefill(a.i32(0), a.ptr<const void>(1), a.i64(2), a.i64(3), a.ptr<const void>(4),
                                   a.i64(5), a.i64(6), a.ptr<const void>(7), a.i64(8), a.i64(9),
                                   a.ptr<const int>(10), a.ptr<const int>(11), a.i32(12), a.i64(13), a.i64(14),
                                   a.i32(15), a.i32(16), a.i32(17), a.real(18), a.i32(19), a.ptr<void>(20),
                                   a.i64(21), a.i64(22), stream);
    default: return frc__fail(FRC_ERR_INVALID, "frc_serving_call: unknown operator");
  }
}
