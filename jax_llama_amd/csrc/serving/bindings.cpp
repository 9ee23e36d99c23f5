// Python bindings of the serving kernels (module jax_llama_amd._C_serving). Thin: validate devices, dtypes, shapes, strides and
// alignment on the host (a wrong shape must never reach a kernel), take raw pointers and launch on the current HIP stream of the
// tensors' device, so hipGraph capture through torch.cuda.graph records these launches.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <map>
#include <unordered_map>
#include <unordered_set>

#include "serving.h"

namespace {

using torch::Tensor;
using OptT = c10::optional<Tensor>;

#define JLA_SV "jax_llama_amd._C_serving: "

hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }

void rc(int r, const char* what) { TORCH_CHECK(r == 0, JLA_SV, what, " failed (code ", r, ")"); }

void on(const Tensor& t, const Tensor& first, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == first.device(), JLA_SV, name, " must be on ", first.device());
}
template <class T>
const T* vec(const OptT& t, const Tensor& first, torch::ScalarType dt, int64_t numel, const char* name) {
  if (!t.has_value()) return nullptr;
  on(*t, first, name);
  TORCH_CHECK(t->scalar_type() == dt && t->is_contiguous() && t->numel() == numel, JLA_SV, name, " must be a contiguous ", dt, " of ",
              numel, " elements");
  return reinterpret_cast<const T*>(t->data_ptr());
}
void aligned(const Tensor& t, int bytes, const char* name) {
  TORCH_CHECK((uintptr_t)t.data_ptr() % bytes == 0, JLA_SV, name, " must start at a multiple of ", bytes, " bytes");
}

// keys or values [N, Hkv, T, 128] whose rows of 128 follow one another; the outer strides
const uint16_t* keys(const Tensor& t, const Tensor& q, int64_t n, int64_t hkv, int64_t len, const char* name, long long* s0, long long* s1) {
  on(t, q, name);
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16 && t.dim() == 4 && t.size(0) == n && t.size(1) == hkv && t.size(2) == len &&
                  t.size(3) == q.size(3),
              JLA_SV, name, " must be bfloat16 [", n, ", ", hkv, ", ", len, ", ", q.size(3), "]");
  TORCH_CHECK(t.stride(3) == 1 && (len == 1 || t.stride(2) == t.size(3)) && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0, JLA_SV, name,
              ": a head's tokens must follow one another, outer strides be multiples of 8");
  aligned(t, 16, name);
  *s0 = t.stride(0);
  *s1 = t.stride(1);
  return reinterpret_cast<const uint16_t*>(t.data_ptr());
}

void prefix_attn(Tensor q, Tensor kp, Tensor vp, Tensor ko, Tensor vo, Tensor slot, OptT prefix_len, OptT prefix_start, OptT prefix_mask,
                 OptT kv_start, Tensor out, OptT out_pack) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 4 && q.scalar_type() == torch::kBFloat16 && q.is_contiguous() && q.size(3) == 128, JLA_SV,
              "prefix_attn: q must be a contiguous bfloat16 GPU tensor [B, S, H, 128]");
  const c10::DeviceGuard guard(q.device());
  TORCH_CHECK(kp.dim() == 4 && ko.dim() == 4, JLA_SV, "prefix_attn: keys are [rows, kv heads, tokens, 128]");
  jla::PrefixAttn a{};
  a.B = q.size(0), a.S = q.size(1), a.H = q.size(2);
  a.G = kp.size(0), a.Hkv = kp.size(1), a.P = kp.size(2), a.T = ko.size(2);
  TORCH_CHECK(a.B > 0 && a.S > 0 && a.H > 0 && a.G > 0 && a.Hkv > 0 && a.P > 0 && a.T > 0 && a.B % a.G == 0 && a.H % a.Hkv == 0, JLA_SV,
              "prefix_attn: rows must be a multiple of the prefixes, heads of the kv heads, and none may be empty");
  TORCH_CHECK((int64_t)a.B * a.S * (a.H / a.Hkv) < (1LL << 31) && q.size(0) * q.size(1) * q.size(2) < (1LL << 33), JLA_SV, "prefix_attn: too many queries");
  a.rep = a.H / a.Hkv, a.n = a.B / a.G;
  aligned(q, 16, "q");
  a.q = reinterpret_cast<const uint16_t*>(q.data_ptr());
  a.kp = keys(kp, q, a.G, a.Hkv, a.P, "prefix keys", &a.kp_g, &a.kp_h);
  a.vp = keys(vp, q, a.G, a.Hkv, a.P, "prefix values", &a.vp_g, &a.vp_h);
  a.ko = keys(ko, q, a.B, a.Hkv, a.T, "own keys", &a.ko_b, &a.ko_h);
  a.vo = keys(vo, q, a.B, a.Hkv, a.T, "own values", &a.vo_b, &a.vo_h);
  a.slot = vec<int32_t>(slot, q, torch::kInt32, 1, "slot");
  a.prefix_len = vec<int32_t>(prefix_len, q, torch::kInt32, a.G, "prefix_len");
  a.prefix_start = vec<int32_t>(prefix_start, q, torch::kInt32, a.G, "prefix_start");
  a.prefix_mask = vec<uint8_t>(prefix_mask, q, torch::kUInt8, (int64_t)a.G * a.P, "prefix_mask");
  a.kv_start = vec<int32_t>(kv_start, q, torch::kInt32, a.B, "kv_start");
  on(out, q, "out");
  TORCH_CHECK(out.scalar_type() == torch::kBFloat16 && out.is_contiguous() && out.numel() == q.numel(), JLA_SV, "prefix_attn: out");
  aligned(out, 8, "out");
  a.out = reinterpret_cast<uint16_t*>(out.data_ptr());
  if (out_pack.has_value()) {
    on(*out_pack, q, "out_pack");
    const int64_t m = q.size(0) * q.size(1), rows = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    TORCH_CHECK(m <= 64 && out_pack->scalar_type() == torch::kBFloat16 && out_pack->is_contiguous() && out_pack->numel() >= rows * a.H * 128, JLA_SV,
                "prefix_attn: out_pack is bfloat16 [padded rows, H * 128] of at most 64 rows");
    aligned(*out_pack, 16, "out_pack");
    a.out_pack = reinterpret_cast<uint16_t*>(out_pack->data_ptr());
  }
  const jla::PrefixPlan p = jla::prefix_attn_plan(a.B, a.S, a.H, a.Hkv, a.G, a.P, a.T);
  // the parts' sums: of this call alone (another stream's or another graph's call has its own)
  Tensor part;
  const long long floats = jla::prefix_attn_workspace(p, a.B, a.S, a.H);
  if (floats > 0) {
    part = torch::empty({floats}, q.options().dtype(torch::kFloat32));
    a.part = part.data_ptr<float>();
  }
  rc(jla::prefix_attn(a, p, stream()), "prefix_attn");
}

const float* number(const py::object& o, const Tensor& x, const char* name, float* value) {
  if (!THPVariable_Check(o.ptr())) {
    *value = o.cast<float>();
    return nullptr;
  }
  return vec<float>(o.cast<Tensor>(), x, torch::kFloat32, x.size(0), name);
}

void process_logits(Tensor x, Tensor out, OptT history, OptT length, OptT start, OptT hmask, int64_t prompt_len, int64_t vocab0,
                    py::object rep, py::object pres, py::object freq, OptT bias, OptT allowed, OptT mask_rows) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.scalar_type() == torch::kFloat32 && (x.size(1) <= 1 || x.stride(1) == 1), JLA_SV,
              "process_logits: logits must be a float32 GPU tensor [B, V] with unit inner stride");
  const c10::DeviceGuard guard(x.device());
  on(out, x, "out");
  TORCH_CHECK(out.scalar_type() == torch::kFloat32 && out.sizes() == x.sizes() && (x.size(1) <= 1 || out.stride(1) == 1), JLA_SV,
              "process_logits: out must be like the logits");
  TORCH_CHECK(x.size(0) < (1LL << 31) && x.size(1) < (1LL << 31) - 65536, JLA_SV, "process_logits: too many rows or columns");
  jla::LogitsArgs a{};
  a.B = x.size(0), a.V = x.size(1);
  a.x = x.data_ptr<float>(), a.out = out.data_ptr<float>();
  a.ldx = x.stride(0), a.ldo = out.stride(0);
  a.vocab0 = vocab0, a.prompt_len = (int)std::min<int64_t>(std::max<int64_t>(prompt_len, 0), 0x7fffffff);
  TORCH_CHECK(vocab0 >= 0 && vocab0 + x.size(1) < (1LL << 31) - 65536, JLA_SV, "process_logits: vocab_start");
  a.rep_rows = number(rep, x, "repetition_penalty", &a.rep);
  a.pres_rows = number(pres, x, "presence_penalty", &a.pres);
  a.freq_rows = number(freq, x, "frequency_penalty", &a.freq);
  if (history.has_value()) {
    on(*history, x, "history");
    TORCH_CHECK(history->scalar_type() == torch::kInt32 && history->dim() == 2 && history->size(0) == a.B && history->size(1) < (1LL << 31) &&
                    (history->size(1) <= 1 || history->stride(1) == 1) && length.has_value(),
                JLA_SV, "process_logits: history must be int32 [B, L] with unit inner stride, and come with its length");
    a.history = history->data_ptr<int32_t>(), a.ldh = history->stride(0), a.L = history->size(1);
    a.length = vec<int32_t>(length, x, torch::kInt32, 1, "length");
    a.start = vec<int32_t>(start, x, torch::kInt32, a.B, "start");
    if (hmask.has_value()) {
      on(*hmask, x, "history_mask");
      TORCH_CHECK(hmask->scalar_type() == torch::kUInt8 && hmask->sizes() == history->sizes() && (a.L <= 1 || hmask->stride(1) == 1), JLA_SV,
                  "process_logits: history_mask must be uint8 of the history's shape");
      a.hmask = hmask->data_ptr<uint8_t>(), a.ldm = hmask->stride(0);
    }
  }
  if (bias.has_value()) {
    on(*bias, x, "bias");
    const bool rows = bias->dim() == 2;
    TORCH_CHECK(bias->scalar_type() == torch::kFloat32 && (rows ? bias->sizes() == x.sizes() : bias->dim() == 1 && bias->size(0) == a.V) &&
                    (a.V <= 1 || bias->stride(-1) == 1),
                JLA_SV, "process_logits: bias must be float32 [V] or [B, V] with unit inner stride");
    a.bias = bias->data_ptr<float>(), a.ldb = rows ? bias->stride(0) : 0;
  }
  if (allowed.has_value()) {
    on(*allowed, x, "allowed");
    TORCH_CHECK(allowed->scalar_type() == torch::kInt32 && allowed->dim() == 2 && allowed->size(0) > 0 && allowed->size(0) < (1LL << 31) &&
                    allowed->size(1) * 32 >= vocab0 + x.size(1) && allowed->stride(1) == 1,
                JLA_SV, "process_logits: allowed must be int32 [masks, words] with a bit for every token id of the columns");
    a.allowed = allowed->data_ptr<int32_t>(), a.ldw = allowed->stride(0), a.n_masks = allowed->size(0);
    a.mask_rows = vec<int32_t>(mask_rows, x, torch::kInt32, a.B, "allowed_rows");
    TORCH_CHECK(a.mask_rows || a.n_masks == 1 || a.n_masks == a.B, JLA_SV, "process_logits: one mask, one per row, or allowed_rows");
  }
  rc(jla::process_logits(a, stream()), "process_logits");
}

// The steps (serving.h) that make row dst[i] row src[i] (-1: zeros), and the first step of each chain. Distinct dst. In place, a row is
// overwritten once nothing waits for what it held; what is left then are cycles, which save their first row. Rows that no step writes
// are read by chains of their own, of at most 8 rows each: their steps need no order.
std::pair<std::vector<int64_t>, std::vector<int64_t>> plan_rows(const std::vector<int64_t>& from, const std::vector<int64_t>& to, bool in_place) {
  TORCH_CHECK_VALUE(from.size() == to.size(), JLA_SV, "plan_rows: as many sources as rows");
  std::vector<int64_t> src, dst, steps, chains{0};
  std::unordered_map<int64_t, int64_t> writer;  // row -> the pair that writes it
  std::unordered_set<int64_t> rows;
  for (size_t i = 0; i < to.size(); ++i) {
    TORCH_CHECK_VALUE(rows.insert(to[i]).second, JLA_SV, "plan_rows: a row is written twice");
    if (in_place && from[i] == to[i]) continue;  // (stays as it is)
    if (in_place) writer[to[i]] = dst.size();
    src.push_back(from[i]), dst.push_back(to[i]);
  }
  const int64_t n = dst.size();
  auto put = [&](int64_t a, int64_t b) { steps.push_back(a), steps.push_back(b); };
  auto end_chain = [&] {
    if ((int64_t)steps.size() / 2 > chains.back()) chains.push_back(steps.size() / 2);
  };
  std::vector<int64_t> source(n, -1), readers(n, 0);  // the pair that writes pair i's source; pairs that read pair i's row
  for (int64_t i = 0; i < n && in_place; ++i) {
    const auto w = writer.find(src[i]);
    if (w != writer.end()) source[i] = w->second, ++readers[w->second];
  }
  std::vector<char> done(n, 0);
  std::vector<int64_t> order(n);
  for (int64_t i = 0; i < n; ++i) order[i] = i;
  std::stable_sort(order.begin(), order.end(), [&](int64_t x, int64_t y) { return src[x] < src[y]; });
  int64_t last = jla::ROW_SAVED, run = 0;
  for (const int64_t i : order) {
    if (readers[i] || source[i] >= 0) continue;
    if (src[i] != last || run == 8) end_chain(), run = 0;
    put(src[i], dst[i]);
    done[i] = 1, last = src[i], ++run;
  }
  end_chain();
  // the others hang together by rows that are both written and read: a chain each
  std::vector<int64_t> group(n);
  for (int64_t i = 0; i < n; ++i) group[i] = i;
  auto root = [&](int64_t i) {
    while (group[i] != i) i = group[i] = group[group[i]];
    return i;
  };
  for (int64_t i = 0; i < n; ++i)
    if (source[i] >= 0) group[root(i)] = root(source[i]);
  std::map<int64_t, std::vector<int64_t>> groups;
  for (int64_t i = 0; i < n; ++i)
    if (!done[i]) groups[root(i)].push_back(i);
  for (const auto& g : groups) {
    std::vector<int64_t> ready;
    for (const int64_t i : g.second)
      if (!readers[i]) ready.push_back(i);
    while (!ready.empty()) {
      const int64_t i = ready.back(), w = source[i];
      ready.pop_back();
      put(src[i], dst[i]);
      done[i] = 1;
      if (w >= 0 && --readers[w] == 0) ready.push_back(w);
    }
    for (const int64_t first : g.second) {  // (one cycle at most: a row has one source)
      if (done[first]) continue;
      put(dst[first], jla::ROW_SAVED);
      int64_t i = first;
      for (; source[i] != first; i = source[i]) put(src[i], dst[i]), done[i] = 1;
      put(jla::ROW_SAVED, dst[i]);
      done[i] = 1;
    }
    end_chain();
  }
  return {steps, chains};
}

// src, dst: int64 [spans, 6] tables on the device (serving.h RowSpan; ops/cache_rows.py makes them)
void copy_rows(Tensor src, Tensor dst, std::vector<int64_t> steps, std::vector<int64_t> chains, OptT long_program, int64_t tokens,
               int64_t widest) {
  static_assert(sizeof(jla::RowSpan) == 48, "a span's layout");
  TORCH_CHECK(src.is_cuda() && src.scalar_type() == torch::kInt64 && src.is_contiguous() && src.dim() == 2 && src.size(1) == 6, JLA_SV,
              "copy_rows: span tables are int64 [spans, 6]");
  const c10::DeviceGuard guard(src.device());
  on(dst, src, "dst");
  TORCH_CHECK(dst.scalar_type() == torch::kInt64 && dst.is_contiguous() && dst.sizes() == src.sizes(), JLA_SV, "copy_rows: equal span tables");
  TORCH_CHECK(steps.size() % 2 == 0 && chains.size() >= 1 && tokens >= 0 && tokens < (1LL << 31), JLA_SV, "copy_rows: program");
  const int64_t n = steps.size() / 2, nc = chains.size() - 1;
  jla::RowProgram p{};
  const int32_t* lp = nullptr;
  if (n > jla::ROW_STEPS) {  // (chains are not empty)
    TORCH_CHECK(long_program.has_value(), JLA_SV, "copy_rows: more steps than an argument holds need long_program");
    lp = vec<int32_t>(long_program, src, torch::kInt32, 2 * n + nc + 1, "long_program");
  } else {
    for (int64_t i = 0; i < 2 * n; ++i) p.step[i] = (int32_t)steps[i];
    for (int64_t i = 0; i <= nc; ++i) p.chain[i] = (uint16_t)chains[i];
  }
  rc(jla::copy_rows(reinterpret_cast<const jla::RowSpan*>(src.data_ptr()), reinterpret_cast<const jla::RowSpan*>(dst.data_ptr()), src.size(0), p,
                    lp, n, nc, tokens, widest, stream()),
     "copy_rows");
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("prefix_attn", &prefix_attn, py::arg("q"), py::arg("kp"), py::arg("vp"), py::arg("ko"), py::arg("vo"), py::arg("slot"),
        py::arg("prefix_len"), py::arg("prefix_start"), py::arg("prefix_mask"), py::arg("kv_start"), py::arg("out"), py::arg("out_pack"));
  m.def("process_logits", &process_logits, py::arg("x"), py::arg("out"), py::arg("history"), py::arg("length"), py::arg("start"),
        py::arg("history_mask"), py::arg("prompt_len"), py::arg("vocab_start"), py::arg("repetition"), py::arg("presence"),
        py::arg("frequency"), py::arg("bias"), py::arg("allowed"), py::arg("allowed_rows"));
  m.def("plan_rows", &plan_rows, py::arg("src"), py::arg("dst"), py::arg("in_place"));
  m.def("copy_rows", &copy_rows, py::arg("src"), py::arg("dst"), py::arg("steps"), py::arg("chains"), py::arg("long_program"),
        py::arg("tokens"), py::arg("widest"));
  m.attr("ROW_STEPS") = (int)jla::ROW_STEPS;
}
