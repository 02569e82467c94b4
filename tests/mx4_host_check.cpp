// The entry points of the operators on 4-bit microscaled matrices with HIP's launch
// functions replaced, for tests/test_mx4_host.py: what tests/operators_host_check.cpp
// does for the 8-bit operators, with its hooks, lines and answers. Beside an
// operator's arguments a line may say `less`, the bytes that the call's workspace
// is smaller than what the query answered.
#define main operators_main
#include "operators_host_check.cpp"
#undef main

namespace {

#define MX4_OPERATOR(name)                                                                          \
  [](auto& q, uint64_t& bytes) { return rns8_mi355x_##name##_workspace(&q, &bytes); },              \
      [&](rns8_context& ctx, auto& q, uint64_t bytes, void* stream) {                               \
        if (bytes) q.workspace = reinterpret_cast<void*>(kWorkspace);                               \
        q.workspace_bytes = bytes - less;                                                           \
        return rns8_mi355x_##name(&ctx, &q, stream);                                                \
      }

bool answer_mx4(const std::string& what, const Values& v) {
  uint64_t less = 0;
  set(v, "less", less);
  if (what == "quantize_mx4" || what == "dequantize_mx4") {
    rns8_mi355x_mx4_args a{};
    SET(rows), SET(cols), SET(x), SET(ldx), SET(q), SET(q_t);
    if (what == "quantize_mx4")
      ask(a, v, OPERATOR_WITHOUT_WORKSPACE(quantize_mx4));
    else
      ask(a, v, OPERATOR_WITHOUT_WORKSPACE(dequantize_mx4));
  } else if (what == "pack_mx4") {
    rns8_mi355x_pack_mx4_args a{};
    SET(rows), SET(cols), SET(data), SET(ldd), SET(scale), SET(lds), SET(q);
    ask(a, v, OPERATOR_WITHOUT_WORKSPACE(pack_mx4));
  } else if (what == "gemm_mx4") {
    rns8_mi355x_gemm_mx4_args a{};
    SET(m), SET(n), SET(k), SET(a), SET(b), SET(bias), SET(out), SET(ldo);
    ask(a, v, MX4_OPERATOR(gemm_mx4));
  } else if (what == "linear_mx4") {
    rns8_mi355x_linear_mx4_args a{};
    SET(m), SET(n), SET(k), SET(x), SET(ldx), SET(w), SET(bias), SET(out), SET(ldo);
    ask(a, v, MX4_OPERATOR(linear_mx4));
  } else if (what == "linear_mx4_backward") {
    rns8_mi355x_linear_mx4_backward_args a{};
    SET(m), SET(n), SET(k), SET(dy), SET(lddy), SET(x), SET(ldx), SET(w_t), SET(dx), SET(lddx), SET(dw), SET(lddw), SET(dbias);
    ask(a, v, MX4_OPERATOR(linear_mx4_backward));
  } else if (what == "experts_mx4") {
    rns8_mi355x_experts_mx4_args a{};
    SET(tokens), SET(experts), SET(width), SET(inner), SET(top), SET(flags), SET(x), SET(ldx), SET(router), SET(ldrouter);
    SET(gate), SET(up), SET(down), SET(out), SET(ldo), SET(ids), SET(weights);
    ask(a, v, MX4_OPERATOR(experts_mx4));
  } else {
    return answer(what, v);
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
    if (!answer_mx4(what, v)) return 2;
  }
  return 0;
}
