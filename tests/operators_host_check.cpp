// Calls the language-model operators' entry points with HIP's launch functions
// replaced by ones that only take notes, for tests/test_operators_host.py: what
// a call would enqueue, without a device. Pointers are addresses that nothing
// reads. Input lines are an operator's name and its arguments by name
// ("linear_i8 m 1 n 0 k 64 ..."), with `stream` for the stream's handle; each
// prints
//
//   <query status> <workspace bytes> <status> <launches> <most workgroups in one> <stream of the last>
//
// where the call is given a workspace of the size that the query answered. The
// context's own stream has the handle 4096. The line "kernels" prints how often
// each kernel of the library was launched so far, and an empty line after them.
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstring>
#include <iostream>
#include <map>
#include <set>
#include <sstream>
#include <string>

#include "handles.hpp"
#include "rns8_mi355x.h"

namespace {
int launches = 0;
uint64_t most_blocks = 0;
hipStream_t last_stream = nullptr;
dim3 grid_of_call, block_of_call;
size_t shared_of_call;
hipStream_t stream_of_call;
// kernels by the host's address of theirs (filled before main, so made on first use)
std::map<const void*, std::string>& kernel_names() {
  static std::map<const void*, std::string> names;
  return names;
}
std::map<std::string, long> kernel_launches;
}  // namespace

extern "C" {
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t stream) {
  grid_of_call = grid;
  block_of_call = block;
  shared_of_call = shared;
  stream_of_call = stream;
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* stream) {
  *grid = grid_of_call;
  *block = block_of_call;
  *shared = shared_of_call;
  *stream = stream_of_call;
  return hipSuccess;
}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
  kernel_names()[host] = name;
}
hipError_t hipLaunchKernel(const void* kernel, dim3 grid, dim3, void**, size_t, hipStream_t stream) {
  ++launches;
  ++kernel_launches[kernel_names()[kernel]];
  const uint64_t blocks = static_cast<uint64_t>(grid.x) * grid.y * grid.z;
  if (blocks > most_blocks) most_blocks = blocks;
  last_stream = stream;
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevice(int* device) {
  *device = 0;
  return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int* value, hipDeviceAttribute_t, int) {
  *value = 256;
  return hipSuccess;
}
}

namespace {

using Values = std::map<std::string, double>;

template <typename T>
void set(const Values& v, const char* name, T& field) {
  const auto it = v.find(name);
  if (it == v.end()) return;
  if constexpr (std::is_pointer_v<T>)
    field = reinterpret_cast<T>(static_cast<uintptr_t>(it->second));
  else
    field = static_cast<T>(it->second);
}
#define SET(name) set(v, #name, a.name)

template <typename A, typename Query, typename Call>
void ask(A& a, const Values& v, Query&& query, Call&& call) {
  a.struct_size = sizeof(A);
  a.abi_version = RNS8_ABI_VERSION;
  SET(dtype);
  uint64_t bytes = 0;
  const rns8_status asked = query(a, bytes);
  rns8_context ctx;
  ctx.stream = reinterpret_cast<hipStream_t>(4096);
  void* stream = nullptr;
  set(v, "stream", stream);
  launches = 0;
  most_blocks = 0;
  last_stream = nullptr;
  const rns8_status status = call(ctx, a, bytes, stream);
  ctx.stream = nullptr;
  std::cout << asked << " " << bytes << " " << status << " " << launches << " " << most_blocks << " "
            << reinterpret_cast<uintptr_t>(last_stream) << "\n";
}

constexpr uintptr_t kWorkspace = uintptr_t{1} << 40;

#define OPERATOR(name)                                                                            \
  [](auto& q, uint64_t& bytes) { return rns8_mi355x_##name##_workspace(&q, &bytes); },            \
      [](rns8_context& ctx, auto& q, uint64_t bytes, void* stream) {                              \
        if (bytes) q.workspace = reinterpret_cast<void*>(kWorkspace);                             \
        q.workspace_bytes = bytes;                                                                \
        return rns8_mi355x_##name(&ctx, &q, stream);                                              \
      }
#define OPERATOR_WITHOUT_WORKSPACE(name)                                        \
  [](auto&, uint64_t&) { return RNS8_SUCCESS; },                                \
      [](rns8_context& ctx, auto& q, uint64_t, void* stream) { return rns8_mi355x_##name(&ctx, &q, stream); }

bool answer(const std::string& what, const Values& v) {
  if (what == "linear_i8") {
    rns8_mi355x_linear_i8_args a{};
    SET(m), SET(n), SET(k), SET(x), SET(ldx), SET(w), SET(ldw), SET(w_scale), SET(bias), SET(out), SET(ldo), SET(x_q);
    SET(ldq), SET(x_scale);
    ask(a, v, OPERATOR(linear_i8));
  } else if (what == "linear_i8_backward") {
    rns8_mi355x_linear_i8_backward_args a{};
    SET(m), SET(n), SET(k), SET(dy), SET(lddy), SET(x_q), SET(ldq), SET(x_scale), SET(w), SET(ldw), SET(w_scale);
    SET(dx), SET(lddx), SET(dw), SET(lddw), SET(dbias);
    ask(a, v, OPERATOR(linear_i8_backward));
  } else if (what == "gemm_i8_scaled") {
    rns8_mi355x_gemm_i8_args a{};
    SET(m), SET(n), SET(k), SET(a), SET(lda), SET(b), SET(ldb), SET(b_layout), SET(out), SET(ldo);
    ask(a, v, OPERATOR(gemm_i8_scaled));
  } else if (what == "quantize_columns") {
    rns8_mi355x_quantize_args a{};
    SET(rows), SET(cols), SET(x), SET(ldx), SET(multiplier), SET(q), SET(ldq), SET(scale), SET(sums);
    ask(a, v, OPERATOR(quantize_columns));
  } else if (what == "quantize_rows") {
    rns8_mi355x_quantize_args a{};
    SET(rows), SET(cols), SET(x), SET(ldx), SET(multiplier), SET(q), SET(ldq), SET(scale);
    ask(a, v, OPERATOR_WITHOUT_WORKSPACE(quantize_rows));
  } else if (what == "block_norm") {
    rns8_mi355x_block_norm_args a{};
    SET(rows), SET(cols), SET(flags), SET(branch_scale), SET(residual_scale), SET(x), SET(ldx), SET(gate), SET(ldgate);
    SET(h), SET(ldh), SET(y), SET(ldy);
    ask(a, v, OPERATOR_WITHOUT_WORKSPACE(block_norm));
  } else if (what == "block_norm_backward") {
    rns8_mi355x_block_norm_backward_args a{};
    SET(rows), SET(cols), SET(flags), SET(branch_scale), SET(residual_scale), SET(x), SET(ldx), SET(gate), SET(ldgate);
    SET(rstd), SET(dy), SET(lddy), SET(dx), SET(lddx), SET(dpre_weight);
    ask(a, v, OPERATOR(block_norm_backward));
  } else if (what == "token_logprobs") {
    rns8_mi355x_logprobs_args a{};
    SET(rows), SET(vocab), SET(logits), SET(ldl), SET(scale), SET(top), SET(lse), SET(top_ids);
    ask(a, v, OPERATOR(token_logprobs));
  } else if (what == "token_logprobs_backward") {
    rns8_mi355x_logprobs_backward_args a{};
    SET(rows), SET(vocab), SET(logits), SET(ldl), SET(targets), SET(scale), SET(lse), SET(dlogp), SET(dlogits), SET(lddl);
    ask(a, v, OPERATOR_WITHOUT_WORKSPACE(token_logprobs_backward));
  } else if (what == "kernels") {
    std::set<std::string> names;
    for (const auto& k : kernel_names()) names.insert(k.second);
    for (const auto& name : names) std::cout << name << " " << kernel_launches[name] << "\n";
    std::cout << "\n";
  } else {
    return false;
  }
  return true;
}

}  // namespace

int main() {
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    std::string what, name;
    double value;
    Values v;
    in >> what;
    while (in >> name >> value) v[name] = value;
    if (!answer(what, v)) return 2;
  }
  return 0;
}
