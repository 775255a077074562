// The plugin's own operators, reached as `stablehlo.custom_call @ryft.<name>` with a backend_config dictionary (the
// typed form, api_version 4): operand and result types, and the config's names and ranges, checked when the program is
// read. The planner turns each call into one step (planner.cc), the kernels are in kernels/k_rope_append.hip,
// k_paged_attention.hip, k_sample.hip, k_int4_matmul.hip and k_tree_accept.hip; their definitions stand beside the argument
// blocks in kernel_abi.h.
#include <cmath>

#include "kernel_abi.h"
#include "mlir_common.h"

namespace ryft {

namespace {

// One call's operands and config under its target's name, for messages that say what was wrong where.
struct Call {
  const Graph& g;
  const Node& n;
  const std::string& target;
  const std::vector<TensorType>& results;

  [[noreturn]] void bad(const std::string& what) const { invalid("custom_call @" + target + ": " + what); }
  const TensorType& operand(size_t i) const { return g.nodes[n.operands[i]].type; }
  void counts(size_t lo, size_t hi, size_t n_results) const {
    if (n.operands.size() != lo && n.operands.size() != hi)
      bad("expected " + std::to_string(lo) + (hi != lo ? " or " + std::to_string(hi) : std::string()) +
          " operands but got " + std::to_string(n.operands.size()));
    if (results.size() != n_results)
      bad("expected " + std::to_string(n_results) + " results but got " + std::to_string(results.size()));
  }
  void is(const char* name, const TensorType& t, DType dt, const std::vector<int64_t>& shape) const {
    const TensorType want{dt, shape};
    if (!(t == want)) bad(std::string(name) + " is " + t.str() + " but must be " + want.str());
  }
  void float16_or_32(const char* name, const TensorType& t) const {
    if (t.dtype != DType::BF16 && t.dtype != DType::F16 && t.dtype != DType::F32)
      unimplemented("custom_call @" + target + ": " + name + " of " + std::string(dtype_name(t.dtype)) +
                    " elements (bf16, f16 and f32 are supported)");
  }
  void rank(const char* name, const TensorType& t, int r) const {
    if (t.rank() != r) bad(std::string(name) + " is " + t.str() + " but must have rank " + std::to_string(r));
  }
  // The config may hold these names and no others.
  void names(std::initializer_list<const char*> known) const {
    for (auto& kv : n.config) {
      bool ok = false;
      for (const char* k : known) ok |= kv.first == k;
      if (!ok) bad("unknown backend_config entry '" + kv.first + "'");
    }
  }
  bool has(const char* k) const { return n.config.count(k) > 0; }
  double number(const char* k, double otherwise, double lo, double hi) const {
    auto it = n.config.find(k);
    const double x = it == n.config.end() ? otherwise : it->second;
    if (!(x >= lo && x <= hi)) bad(std::string(k) + " = " + std::to_string(x) + " is out of range");
    return x;
  }
  void whole(const char* k, double x) const {
    if (x != std::floor(x)) bad(std::string(k) + " must be a whole number");
  }
};

constexpr int64_t kMaxHeadDim = 256;
constexpr double kFloatMax = 0x1.fffffefffffffp127;  // the largest that rounds to a finite f32

void check_cache(const Call& c, const TensorType& kc, const TensorType& vc, DType dt, int64_t hkv, int64_t d) {
  c.rank("the key cache", kc, 4);
  if (kc.dtype != dt || kc.shape[3] != d || (hkv >= 0 && kc.shape[1] != hkv))
    c.bad("the key cache is " + kc.str() + " but must be [pages, " + (hkv >= 0 ? std::to_string(hkv) : "key heads") +
          ", page size, " + std::to_string(d) + "] of " + dtype_name(dt));
  if (kc.shape[1] < 1 || kc.shape[2] < 1) c.bad("the cache's key heads and page size must be at least 1");
  if (kc.shape[1] > (1 << 16) || kc.shape[2] > (1 << 20) || kc.shape[0] > INT32_MAX)
    c.bad("the key cache's extents are out of range");
  if (!(vc == kc)) c.bad("the value cache is " + vc.str() + " but must be " + kc.str());
}

// (q, k, v, positions, slots, inv_freq, k_cache, v_cache[, q_weight, k_weight]) -> (q, k_cache, v_cache)
void check_rope_append(const Call& c, std::map<std::string, double>* config) {
  c.counts(8, 10, 3);
  c.names({"eps", "interleaved", "magnitude"});
  const TensorType &q = c.operand(0), &k = c.operand(1), &f = c.operand(5), &kc = c.operand(6);
  c.float16_or_32("q", q);
  c.rank("q", q, 3);
  c.rank("k", k, 3);
  const int64_t T = q.shape[0], hkv = k.shape[1], d = q.shape[2];
  if (q.shape[1] < 1 || q.shape[1] > (1 << 16) || hkv < 1) c.bad("q and k need at least one head");
  if (d < 1 || d > kMaxHeadDim) c.bad("head dim " + std::to_string(d) + " is out of range (1 to 256)");
  if (T > INT32_MAX) c.bad("too many tokens");
  c.is("k", k, q.dtype, {T, hkv, d});
  c.is("v", c.operand(2), q.dtype, {T, hkv, d});
  c.is("positions", c.operand(3), DType::S32, {T});
  c.is("slots", c.operand(4), DType::S32, {T});
  c.rank("inv_freq", f, 1);
  c.is("inv_freq", f, DType::F32, {f.shape[0]});
  if (2 * f.shape[0] > d) c.bad("inv_freq has " + std::to_string(f.shape[0]) + " entries: at most half the head dim");
  check_cache(c, kc, c.operand(7), q.dtype, hkv, d);
  if (c.n.operands.size() == 10) {
    c.is("q_weight", c.operand(8), q.dtype, {d});
    c.is("k_weight", c.operand(9), q.dtype, {d});
  } else if (c.has("eps")) {
    c.bad("eps needs the norm weights");
  }
  c.is("result 0", c.results[0], q.dtype, q.shape);
  c.is("result 1", c.results[1], kc.dtype, kc.shape);
  c.is("result 2", c.results[2], kc.dtype, kc.shape);
  (*config)["eps"] = c.number("eps", 1e-6, 0, 1e6);
  (*config)["interleaved"] = c.number("interleaved", 0, 0, 1);
  (*config)["magnitude"] = c.number("magnitude", 1.0, -1e6, 1e6);
}

// The operands that paged_attention and tree_attention share, the result and their config.
void check_attention(const Call& c, std::map<std::string, double>* config) {
  const TensorType &q = c.operand(0), &kc = c.operand(1), &tab = c.operand(3), &len = c.operand(5);
  c.float16_or_32("q", q);
  c.rank("q", q, 3);
  const int64_t T = q.shape[0], hq = q.shape[1], d = q.shape[2];
  if (hq < 1 || hq > 65535) c.bad("q needs 1 to 65535 heads");
  if (d < 1 || d > kMaxHeadDim) c.bad("head dim " + std::to_string(d) + " is out of range (1 to 256)");
  if (T > INT32_MAX) c.bad("too many tokens");
  check_cache(c, kc, c.operand(2), q.dtype, -1, d);
  if (hq % kc.shape[1]) c.bad(std::to_string(hq) + " query heads are no multiple of " + std::to_string(kc.shape[1]) + " key heads");
  c.rank("page_table", tab, 2);
  c.rank("lengths", len, 1);
  const int64_t B = len.shape[0];
  c.is("page_table", tab, DType::S32, {B, tab.shape[1]});
  c.is("starts", c.operand(4), DType::S32, {B + 1});
  c.is("lengths", len, DType::S32, {B});
  if (B > (1 << 20) || tab.shape[1] * kc.shape[2] > INT32_MAX - 65536) c.bad("too many sequences, or too long ones");
  c.is("the result", c.results[0], q.dtype, q.shape);
  (*config)["scale"] = c.number("scale", 1.0 / std::sqrt((double)d), -kFloatMax, kFloatMax);
  (*config)["softcap"] = c.number("softcap", 0, 0, kFloatMax);
  (*config)["window"] = c.number("window", 0, 0, INT32_MAX);
  c.whole("window", (*config)["window"]);
}

// (q, k_cache, v_cache, page_table, starts, lengths[, slopes]) -> o
void check_paged_attention(const Call& c, std::map<std::string, double>* config) {
  c.counts(6, 7, 1);
  c.names({"scale", "softcap", "window", "causal"});
  check_attention(c, config);
  if (c.n.operands.size() == 7) c.is("slopes", c.operand(6), DType::F32, {c.operand(0).shape[1]});
  (*config)["causal"] = c.number("causal", 1, 0, 1);
}

// (q, k_cache, v_cache, page_table, starts, lengths, visible) -> o
void check_tree_attention(const Call& c, std::map<std::string, double>* config) {
  c.counts(7, 7, 1);
  c.names({"scale", "softcap", "window"});
  check_attention(c, config);
  const TensorType& vis = c.operand(6);
  c.rank("visible", vis, 2);
  c.is("visible", vis, DType::S32, {c.operand(0).shape[0], vis.shape[1]});
  if (vis.shape[1] < 1 || vis.shape[1] > (1 << 16)) c.bad("visible needs 1 to 65536 words a token");
  (*config)["causal"] = 0;
}

// (logits, temperature, top_k, top_p, min_p, uniform) -> (token, logprob)
void check_sample(const Call& c, std::map<std::string, double>* config) {
  c.counts(6, 6, 2);
  c.names({});
  const TensorType& x = c.operand(0);
  c.float16_or_32("logits", x);
  c.rank("logits", x, 2);
  const int64_t B = x.shape[0], V = x.shape[1];
  if (V < 1 || V > (1 << 24)) c.bad("a vocabulary of " + std::to_string(V) + " is out of range (1 to 2^24)");
  if (B > (1 << 20)) c.bad("too many rows");
  const char* names[] = {"", "temperature", "top_k", "top_p", "min_p", "uniform"};
  for (int i = 1; i < 6; ++i) c.is(names[i], c.operand(i), i == 2 ? DType::S32 : DType::F32, {B});
  c.is("result 0", c.results[0], DType::S32, {B});
  c.is("result 1", c.results[1], DType::F32, {B});
}

// (x, weight, scale[, zero]) -> y
void check_int4_matmul(const Call& c, std::map<std::string, double>*) {
  c.counts(3, 4, 1);
  c.names({});
  const TensorType &x = c.operand(0), &w = c.operand(1), &s = c.operand(2), &y = c.results[0];
  c.float16_or_32("x", x);
  c.float16_or_32("scale", s);
  c.float16_or_32("the result", y);
  c.rank("x", x, 2);
  c.rank("weight", w, 2);
  c.rank("scale", s, 2);
  const int64_t T = x.shape[0], K = x.shape[1], N = w.shape[0], groups = s.shape[1];
  if (K < 2 || K % 2 || K > (1 << 24)) c.bad("x has rows of " + std::to_string(K) + " values: an even number up to 2^24 is needed");
  if (N < 1 || N > (1 << 24)) c.bad("a weight of " + std::to_string(N) + " rows is out of range (1 to 2^24)");
  if (T > INT32_MAX) c.bad("too many rows");
  c.is("weight", w, DType::U8, {N, K / 2});
  c.is("scale", s, s.dtype, {N, groups});
  if (s.dtype != x.dtype && s.dtype != DType::F32) c.bad("scale is " + s.str() + " but must have x's element type or f32");
  if (y.dtype != x.dtype && y.dtype != DType::F32) c.bad("the result is " + y.str() + " but must have x's element type or f32");
  if (groups < 1 || K % groups || K / groups % 2)
    c.bad("rows of " + std::to_string(K) + " values are not cut into " + std::to_string(groups) + " groups of an even number of values");
  if (c.n.operands.size() == 4) c.is("zero", c.operand(3), DType::U8, s.shape);
  c.is("the result", y, y.dtype, {T, N});
}

// (tokens, parents, targets, slots, starts, caches...) -> (counts, emitted, path, caches...)
void check_tree_accept(const Call& c, std::map<std::string, double>*) {
  const size_t n = c.n.operands.size() < 5 ? 0 : c.n.operands.size() - 5;
  if (n > (size_t)kMaxTreeCaches) c.bad(std::to_string(n) + " caches: at most " + std::to_string(kMaxTreeCaches));
  c.counts(5 + n, 5 + n, 3 + n);
  c.names({});
  const TensorType &tok = c.operand(0), &st = c.operand(4);
  c.rank("tokens", tok, 1);
  c.rank("starts", st, 1);
  const int64_t T = tok.shape[0], B = st.shape[0] - 1;
  // (the kernel counts nodes in 32 bits, a workgroup's 256 at a time)
  if (B < 0 || B > (1 << 20) || T > (1 << 30)) c.bad("too many tokens or sequences, or no starts");
  const char* names[] = {"tokens", "parents", "targets", "slots"};
  for (int i = 0; i < 4; ++i) c.is(names[i], c.operand(i), DType::S32, {T});
  c.is("starts", st, DType::S32, {B + 1});
  for (size_t i = 0; i < n; ++i) {
    const TensorType& kc = c.operand(5 + i);
    if (i == 0) {
      c.float16_or_32("the cache", kc);
      c.rank("the cache", kc, 4);
      if (kc.shape[3] < 1 || kc.shape[3] > kMaxHeadDim) c.bad("head dim " + std::to_string(kc.shape[3]) + " is out of range (1 to 256)");
      check_cache(c, kc, kc, kc.dtype, -1, kc.shape[3]);
    }
    c.is("a cache", kc, c.operand(5).dtype, c.operand(5).shape);
    c.is("a cache's result", c.results[3 + i], kc.dtype, kc.shape);
  }
  c.is("result 0", c.results[0], DType::S32, {B});
  c.is("result 1", c.results[1], DType::S32, {T});
  c.is("result 2", c.results[2], DType::S32, {T});
}

typedef void (*Check)(const Call&, std::map<std::string, double>*);
Check check_of(const std::string& target) {
  if (target == "ryft.rope_append") return check_rope_append;
  if (target == "ryft.paged_attention") return check_paged_attention;
  if (target == "ryft.sample") return check_sample;
  if (target == "ryft.tree_attention") return check_tree_attention;
  if (target == "ryft.int4_matmul") return check_int4_matmul;
  if (target == "ryft.tree_accept") return check_tree_accept;
  unimplemented("custom_call target '" + target + "' is not provided by the MI355X plugin");
}

}  // namespace

void custom_call_target(const std::string& target) { check_of(target); }

std::vector<Node> custom_call_nodes(const Graph& g, const Node& proto, const std::string& target,
                                    const std::vector<TensorType>& results) {
  const Call c{g, proto, target, results};
  std::map<std::string, double> config;
  check_of(target)(c, &config);
  std::vector<Node> nodes;
  for (size_t i = 0; i < results.size(); ++i) {
    Node m = proto;
    m.op = Op::CustomCall;
    m.type = results[i];
    m.call_target = target;
    m.config = config;
    m.call = (int)g.nodes.size();  // (the op's first node: no other op has it)
    m.result_index = (int)i;
    nodes.push_back(std::move(m));
  }
  return nodes;
}

}  // namespace ryft
