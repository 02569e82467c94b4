// Argument checks and the order of a call that the operators' C entry points share.
#pragma once

#include <cstdint>

#include "contract.hpp"
#include "handles.hpp"
#include "operators.hpp"

namespace rns8x {

constexpr int64_t kMaxSize = 0x7FFFFFFF;

inline bool known_type(uint32_t dtype) { return dtype <= RNS8_MI355X_BF16; }

inline uint64_t element_size(uint32_t dtype) { return dtype == RNS8_MI355X_F32 ? 4u : 2u; }

// A rows x cols operand of elements of `size` bytes: a stride that holds a
// row, offsets that fit 64 bits, a pointer aligned to its elements. An operand
// without elements may be NULL.
inline bool operand_ok(const void* p, int64_t rows, int64_t cols, int64_t ld, uint64_t size) {
  if (ld < cols) return false;
  if (rows == 0 || cols == 0) return true;
  return p && reinterpret_cast<uintptr_t>(p) % size == 0 &&
         valid_access(rows, cols, ld) && rows <= INT64_MAX / static_cast<int64_t>(size) / ld;
}
inline bool optional_ok(const void* p, int64_t rows, int64_t cols, int64_t ld, uint64_t size) {
  return !p || operand_ok(p, rows, cols, ld, size);
}
// An output may be an input itself, row for row; rows at another stride would
// overwrite inputs that are still to be read.
inline bool in_place_ok(const void* in, int64_t ldin, const void* out, int64_t ldout, int64_t rows) {
  return in != out || !out || ldin == ldout || rows < 2;
}
inline bool floats_ok(const void* p, int64_t count) { return operand_ok(p, 1, count, count, sizeof(float)); }

inline rns8_status check_workspace(const void* p, uint64_t have, uint64_t need) {
  if (need == 0) return RNS8_SUCCESS;
  if (have < need) return RNS8_WORKSPACE_TOO_SMALL;
  return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 ? RNS8_SUCCESS : RNS8_INVALID_ARGUMENT;
}

inline rns8_status launched(hipError_t e) {
  if (e == hipSuccess) return RNS8_SUCCESS;
  return e == hipErrorInvalidValue ? RNS8_UNSUPPORTED_BACKEND : RNS8_BACKEND_FAILURE;
}

template <typename A>
bool header_ok(const A* a) {
  return a && valid_abi(a->struct_size, a->abi_version, sizeof(A)) && known_type(a->dtype);
}

// check -> size of the workspace -> `enqueue(stream)` on the context's device
template <typename A, typename Check, typename Size, typename Enqueue>
rns8_status run_operator(rns8_context* ctx, const A* args, void* stream, Check&& check, Size&& size,
                         Enqueue&& enqueue) {
  return guard([&]() -> rns8_status {
    if (!ctx || !header_ok(args)) return RNS8_INVALID_ARGUMENT;
    rns8_status st = check(*args);
    if (st != RNS8_SUCCESS) return st;
    st = size(*args);
    if (st != RNS8_SUCCESS) return st;
    if (hipSetDevice(ctx->device_id) != hipSuccess) return RNS8_BACKEND_FAILURE;
    return launched(enqueue(*args, pick_stream(*ctx, stream)));
  });
}

template <typename A, typename Check, typename Size>
rns8_status workspace_query(const A* args, uint64_t* bytes, Check&& check, Size&& size) {
  return guard([&]() -> rns8_status {
    if (!bytes || !header_ok(args)) return RNS8_INVALID_ARGUMENT;
    *bytes = 0;
    const rns8_status st = check(*args);
    if (st == RNS8_SUCCESS) *bytes = size(*args);
    return st;
  });
}

template <typename A>
rns8_status no_workspace(const A&) {
  return RNS8_SUCCESS;
}

}  // namespace rns8x
