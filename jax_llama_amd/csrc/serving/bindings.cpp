// Python bindings of the serving kernels (module jax_llama_amd._C_serving). Thin: validate devices, dtypes, shapes, strides and
// alignment on the host (a wrong shape must never reach a kernel), take raw pointers and launch on the current HIP stream of the
// tensors' device, so hipGraph capture through torch.cuda.graph records these launches.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
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
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == first.device(), JLA_SV, name, " must be on ", first.device());
}
template <class T>
const T* vec(const OptT& t, const Tensor& first, torch::ScalarType dt, int64_t numel, const char* name) {
  if (!t.has_value()) return nullptr;
  on(*t, first, name);
  TORCH_CHECK_VALUE(t->scalar_type() == dt && t->is_contiguous() && t->numel() == numel, JLA_SV, name, " must be a contiguous ", dt, " of ",
              numel, " elements");
  return reinterpret_cast<const T*>(t->data_ptr());
}
void aligned(const Tensor& t, int bytes, const char* name) {
  TORCH_CHECK_VALUE((uintptr_t)t.data_ptr() % bytes == 0, JLA_SV, name, " must start at a multiple of ", bytes, " bytes");
}

// keys or values [N, Hkv, T, 128] whose rows of 128 follow one another; the outer strides
const uint16_t* keys(const Tensor& t, const Tensor& q, int64_t n, int64_t hkv, int64_t len, const char* name, long long* s0, long long* s1) {
  on(t, q, name);
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kBFloat16 && t.dim() == 4 && t.size(0) == n && t.size(1) == hkv && t.size(2) == len &&
                  t.size(3) == q.size(3),
              JLA_SV, name, " must be bfloat16 [", n, ", ", hkv, ", ", len, ", ", q.size(3), "]");
  TORCH_CHECK_VALUE(t.stride(3) == 1 && (len == 1 || t.stride(2) == t.size(3)) && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0, JLA_SV, name,
              ": a head's tokens must follow one another, outer strides be multiples of 8");
  aligned(t, 16, name);
  *s0 = t.stride(0);
  *s1 = t.stride(1);
  return reinterpret_cast<const uint16_t*>(t.data_ptr());
}

// a device int32[1], or a number (returned in *value)
const int32_t* place(const py::object& o, const Tensor& first, const char* name, int64_t* value) {
  if (!THPVariable_Check(o.ptr())) {
    *value = o.cast<int64_t>();
    return nullptr;
  }
  *value = 0;
  return vec<int32_t>(o.cast<Tensor>(), first, torch::kInt32, 1, name);
}

Tensor prefix_attn(Tensor q, Tensor kp, Tensor vp, Tensor ko, Tensor vo, py::object slot, OptT prefix_len, OptT prefix_start, OptT prefix_mask,
                   OptT kv_start, OptT out_pack) {
  TORCH_CHECK_VALUE(q.is_cuda() && q.dim() == 4 && q.scalar_type() == torch::kBFloat16 && q.is_contiguous() && q.size(3) == 128, JLA_SV,
              "prefix_attn: q must be a contiguous bfloat16 GPU tensor [B, S, H, 128]");
  const c10::DeviceGuard guard(q.device());
  TORCH_CHECK_VALUE(kp.dim() == 4 && ko.dim() == 4, JLA_SV, "prefix_attn: keys are [rows, kv heads, tokens, 128]");
  jla::PrefixAttn a{};
  a.B = q.size(0), a.S = q.size(1), a.H = q.size(2);
  a.G = kp.size(0), a.Hkv = kp.size(1), a.P = kp.size(2), a.T = ko.size(2);
  TORCH_CHECK_VALUE(a.B > 0 && a.S > 0 && a.H > 0 && a.G > 0 && a.Hkv > 0 && a.P > 0 && a.T > 0 && a.B % a.G == 0 && a.H % a.Hkv == 0, JLA_SV,
              "prefix_attn: rows must be a multiple of the prefixes, heads of the kv heads, and none may be empty");
  TORCH_CHECK_VALUE((int64_t)a.B * a.S * (a.H / a.Hkv) < (1LL << 31) && q.size(0) * q.size(1) * q.size(2) < (1LL << 33), JLA_SV, "prefix_attn: too many queries");
  a.rep = a.H / a.Hkv, a.n = a.B / a.G;
  aligned(q, 16, "q");
  a.q = reinterpret_cast<const uint16_t*>(q.data_ptr());
  a.kp = keys(kp, q, a.G, a.Hkv, a.P, "prefix keys", &a.kp_g, &a.kp_h);
  a.vp = keys(vp, q, a.G, a.Hkv, a.P, "prefix values", &a.vp_g, &a.vp_h);
  a.ko = keys(ko, q, a.B, a.Hkv, a.T, "own keys", &a.ko_b, &a.ko_h);
  a.vo = keys(vo, q, a.B, a.Hkv, a.T, "own values", &a.vo_b, &a.vo_h);
  int64_t slot0;
  a.slot = place(slot, q, "slot0", &slot0);
  TORCH_CHECK_VALUE(a.slot || (slot0 >= 0 && slot0 + a.S <= a.T), JLA_SV, "own slots ", slot0, " .. ", slot0 + a.S - 1, " lie outside the cache's ", a.T);
  a.slot0 = (int)slot0;
  a.prefix_len = vec<int32_t>(prefix_len, q, torch::kInt32, a.G, "prefix_len");
  a.prefix_start = vec<int32_t>(prefix_start, q, torch::kInt32, a.G, "prefix_start");
  a.prefix_mask = vec<uint8_t>(prefix_mask, q, torch::kUInt8, (int64_t)a.G * a.P, "prefix_mask");
  a.kv_start = vec<int32_t>(kv_start, q, torch::kInt32, a.B, "kv_start");
  const Tensor out = torch::empty({q.size(0) * q.size(1), q.size(2) * q.size(3)}, q.options());
  a.out = reinterpret_cast<uint16_t*>(out.data_ptr());
  if (out_pack.has_value()) {
    on(*out_pack, q, "out_pack");
    const int64_t m = q.size(0) * q.size(1), rows = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    TORCH_CHECK_VALUE(m <= 64 && out_pack->scalar_type() == torch::kBFloat16 && out_pack->is_contiguous() && out_pack->numel() >= rows * a.H * 128, JLA_SV,
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
  return out;
}

const float* number(const py::object& o, const Tensor& x, const char* name, float* value) {
  if (!THPVariable_Check(o.ptr())) {
    *value = o.cast<float>();
    return nullptr;
  }
  return vec<float>(o.cast<Tensor>(), x, torch::kFloat32, x.size(0), name);
}

Tensor process_logits(Tensor x, OptT into, OptT history, py::object length, OptT start, OptT hmask, int64_t prompt_len, int64_t vocab0,
                    py::object rep, py::object pres, py::object freq, OptT bias, OptT allowed, OptT mask_rows) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() == 2 && x.scalar_type() == torch::kFloat32 && (x.size(1) <= 1 || x.stride(1) == 1), JLA_SV,
              "process_logits: logits must be a float32 GPU tensor [B, V] with unit inner stride");
  const c10::DeviceGuard guard(x.device());
  const Tensor out = into.has_value() ? *into : torch::empty(x.sizes(), x.options());
  if (into.has_value()) {
    on(out, x, "out");
    TORCH_CHECK_VALUE(out.scalar_type() == torch::kFloat32 && out.sizes() == x.sizes() && (x.size(1) <= 1 || out.stride(1) == 1) &&
                          (x.size(0) <= 1 || out.stride(0) >= x.size(1)),
                      JLA_SV, "process_logits: out must be like the logits, its rows apart");
    const char *x0 = (const char*)x.data_ptr(), *o0 = (const char*)out.data_ptr();
    const bool same = x0 == o0 && (x.size(0) <= 1 || x.stride(0) == out.stride(0));
    const bool apart = !x.numel() || x0 + 4 * ((x.size(0) - 1) * x.stride(0) + x.size(1)) <= o0 || o0 + 4 * ((x.size(0) - 1) * out.stride(0) + x.size(1)) <= x0;
    TORCH_CHECK_VALUE(same || apart, JLA_SV, "process_logits: out is the logits or shares nothing with them");
  }
  TORCH_CHECK_VALUE(x.size(0) < (1LL << 31) && x.size(1) < (1LL << 31) - 65536, JLA_SV, "process_logits: too many rows or columns");
  jla::LogitsArgs a{};
  a.B = x.size(0), a.V = x.size(1);
  a.x = x.data_ptr<float>(), a.out = out.data_ptr<float>();
  a.ldx = x.stride(0), a.ldo = out.stride(0);
  a.vocab0 = vocab0, a.prompt_len = (int)std::min<int64_t>(std::max<int64_t>(prompt_len, 0), 0x7fffffff);
  TORCH_CHECK_VALUE(vocab0 >= 0 && vocab0 + x.size(1) < (1LL << 31) - 65536, JLA_SV, "process_logits: vocab_start");
  a.rep = 1.f;
  a.rep_rows = number(rep, x, "repetition_penalty", &a.rep);
  a.pres_rows = number(pres, x, "presence_penalty", &a.pres);
  a.freq_rows = number(freq, x, "frequency_penalty", &a.freq);
  TORCH_CHECK_VALUE(std::isfinite(a.rep) && a.rep > 0.f && std::isfinite(a.pres) && std::isfinite(a.freq) && prompt_len >= 0, JLA_SV,
                    "process_logits: a repetition penalty above 0, finite penalties, prompt_len from 0 on");
  const bool penalised = a.rep_rows || a.pres_rows || a.freq_rows || a.rep != 1.f || a.pres != 0.f || a.freq != 0.f;
  TORCH_CHECK_VALUE(!penalised || (history.has_value() && !length.is_none()), JLA_SV, "process_logits: penalties need the history and its length");
  if (penalised) {
    on(*history, x, "history");
    TORCH_CHECK_VALUE(history->scalar_type() == torch::kInt32 && history->dim() == 2 && history->size(0) == a.B && history->size(1) < (1LL << 31) &&
                    (history->size(1) <= 1 || history->stride(1) == 1),
                JLA_SV, "process_logits: history must be int32 [B, L] with unit inner stride");
    a.history = history->data_ptr<int32_t>(), a.ldh = history->stride(0), a.L = history->size(1);
    int64_t length0;
    a.length = place(length, x, "length", &length0);
    TORCH_CHECK_VALUE(a.length || (length0 >= 0 && length0 <= a.L), JLA_SV, "process_logits: length ", length0, " of a history of ", a.L);
    a.length0 = (int)length0;
    a.start = vec<int32_t>(start, x, torch::kInt32, a.B, "start");
    if (hmask.has_value()) {
      on(*hmask, x, "history_mask");
      TORCH_CHECK_VALUE(hmask->scalar_type() == torch::kUInt8 && hmask->sizes() == history->sizes() && (a.L <= 1 || hmask->stride(1) == 1), JLA_SV,
                  "process_logits: history_mask must be uint8 of the history's shape");
      a.hmask = hmask->data_ptr<uint8_t>(), a.ldm = hmask->stride(0);
    }
  }
  if (bias.has_value()) {
    on(*bias, x, "bias");
    const bool rows = bias->dim() == 2;
    TORCH_CHECK_VALUE(bias->scalar_type() == torch::kFloat32 && (rows ? bias->sizes() == x.sizes() : bias->dim() == 1 && bias->size(0) == a.V) &&
                    (a.V <= 1 || bias->stride(-1) == 1),
                JLA_SV, "process_logits: bias must be float32 [V] or [B, V] with unit inner stride");
    a.bias = bias->data_ptr<float>(), a.ldb = rows ? bias->stride(0) : 0;
  }
  if (allowed.has_value()) {
    on(*allowed, x, "allowed");
    TORCH_CHECK_VALUE(allowed->scalar_type() == torch::kInt32 && allowed->dim() == 2 && allowed->size(0) > 0 && allowed->size(0) < (1LL << 31) &&
                    allowed->size(1) * 32 >= vocab0 + x.size(1) && allowed->stride(1) == 1,
                JLA_SV, "process_logits: allowed must be int32 [masks, words] with a bit for every token id of the columns");
    a.allowed = allowed->data_ptr<int32_t>(), a.ldw = allowed->stride(0), a.n_masks = allowed->size(0);
    a.mask_rows = vec<int32_t>(mask_rows, x, torch::kInt32, a.B, "allowed_rows");
    TORCH_CHECK_VALUE(a.mask_rows || a.n_masks == 1 || a.n_masks == a.B, JLA_SV, "process_logits: one mask, one per row, or allowed_rows");
  }
  TORCH_CHECK_VALUE(allowed.has_value() || !mask_rows.has_value(), JLA_SV, "process_logits: allowed_rows without allowed");
  rc(jla::process_logits(a, stream()), "process_logits");
  return out;
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

bool capturing(hipStream_t st) {
  hipStreamCaptureStatus c = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(st, &c) == hipSuccess && c != hipStreamCaptureStatusNone;
}

// What a cache's rows are made of (ops/cache_rows.py RowLayout): eight numbers a span, as serving.h has them
struct RowLayout {
  std::vector<jla::RowSpan> spans;
  int64_t rows;
  c10::Device device;
  Tensor table;

  RowLayout(const std::vector<int64_t>& words, int64_t rows, Tensor like) : rows(rows), device(like.device()) {
    static_assert(sizeof(jla::RowSpan) == 64, "eight numbers a span");
    TORCH_CHECK_VALUE(like.is_cuda() && words.size() % 8 == 0, JLA_SV, "RowLayout: eight numbers a span of GPU tensors");
    const auto* w = reinterpret_cast<const jla::RowSpan*>(words.data());
    spans.assign(w, w + words.size() / 8);
  }

  // row dst[i] of `to` becomes row src[i] (-1: zeros): the first `tokens` tokens, and what has none
  void copy(RowLayout& to, const std::vector<int64_t>& src, const std::vector<int64_t>& dst, int64_t tokens) {
    TORCH_CHECK_VALUE(spans.size() == to.spans.size() && device == to.device, JLA_SV, "copy_rows: the caches are laid out differently");
    TORCH_CHECK_VALUE(src.size() == dst.size() && tokens >= 0 && tokens < (1LL << 31), JLA_SV, "copy_rows: as many sources as rows");
    for (const int64_t r : src) TORCH_CHECK_VALUE(r >= -1 && r < rows, JLA_SV, "copy_rows: source row ", r, " of a cache of ", rows);
    for (const int64_t r : dst) TORCH_CHECK_VALUE(r >= 0 && r < to.rows, JLA_SV, "copy_rows: row ", r, " of a cache of ", to.rows);
    const auto plan = plan_rows(src, dst, this == &to);
    const int64_t n = plan.first.size() / 2, nc = plan.second.size() - 1;
    if (!n || spans.empty()) return;
    const c10::DeviceGuard guard(device);
    const hipStream_t st = stream();
    long long blocks = 0;
    for (size_t i = 0; i < spans.size(); ++i) {
      const jla::RowSpan &a = spans[i], &b = to.spans[i];
      TORCH_CHECK_VALUE(a.layers == b.layers && a.runs == b.runs && a.token_bytes == b.token_bytes && a.fixed_bytes == b.fixed_bytes, JLA_SV,
                        "copy_rows: the caches are laid out differently");
      const long long bytes = a.token_bytes ? a.token_bytes * tokens : a.fixed_bytes;
      blocks = std::max(blocks, a.layers * a.runs * ((bytes + (1 << 14) - 1) >> 14));
    }
    jla::RowProgram p{};
    Tensor program;
    if (n > jla::ROW_STEPS) {  // (chains are not empty)
      TORCH_CHECK(!capturing(st), JLA_SV, "copies to more than some ", jla::ROW_STEPS, " rows cannot be captured");
      std::vector<int32_t> all(plan.first.begin(), plan.first.end());
      all.insert(all.end(), plan.second.begin(), plan.second.end());
      const Tensor host = torch::empty({(int64_t)all.size()}, torch::TensorOptions().dtype(torch::kInt32).pinned_memory(true));
      std::copy(all.begin(), all.end(), host.data_ptr<int32_t>());
      program = host.to(device, /*non_blocking=*/true);
    } else {
      std::copy(plan.first.begin(), plan.first.end(), p.step);
      std::copy(plan.second.begin(), plan.second.end(), p.chain);
    }
    const bool tables = spans.size() > (size_t)jla::ROW_SPANS;
    if (!tables) {
      std::copy(spans.begin(), spans.end(), p.src);
      std::copy(to.spans.begin(), to.spans.end(), p.dst);
    }
    rc(jla::copy_rows(p, program.defined() ? program.data_ptr<int32_t>() : nullptr, tables ? on_device(st) : nullptr, tables ? to.on_device(st) : nullptr,
                      spans.size(), n, nc, tokens, blocks, st),
       "copy_rows");
  }

  const jla::RowSpan* on_device(hipStream_t st) {
    if (!table.defined()) {
      TORCH_CHECK(!capturing(st), JLA_SV, "the first copy of a cache's rows cannot be captured: make one before");
      const int64_t n = spans.size() * 8;
      table = torch::from_blob(spans.data(), {n}, torch::kInt64).to(device);
    }
    return reinterpret_cast<const jla::RowSpan*>(table.data_ptr());
  }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("prefix_attn", &prefix_attn, py::arg("q"), py::arg("kp"), py::arg("vp"), py::arg("ko"), py::arg("vo"), py::arg("slot"),
        py::arg("prefix_len"), py::arg("prefix_start"), py::arg("prefix_mask"), py::arg("kv_start"), py::arg("out_pack"));
  // the way a call of these sizes goes: in one launch, by row or by group, with a join or without
  m.def("prefix_plan", [](int b, int s, int h, int hkv, int g, int p, int t) {
    const jla::PrefixPlan plan = jla::prefix_attn_plan(b, s, h, hkv, g, p, t);
    return std::string(plan.brief ? "short" : plan.by_row ? "row" : "group") + (!plan.brief && plan.parts() > 1 ? "+join" : "");
  });
  m.def("process_logits", &process_logits, py::arg("x"), py::arg("out"), py::arg("history"), py::arg("length"), py::arg("start"),
        py::arg("history_mask"), py::arg("prompt_len"), py::arg("vocab_start"), py::arg("repetition"), py::arg("presence"),
        py::arg("frequency"), py::arg("bias"), py::arg("allowed"), py::arg("allowed_rows"));
  m.def("plan_rows", &plan_rows, py::arg("src"), py::arg("dst"), py::arg("in_place"));
  py::class_<RowLayout>(m, "RowLayout")
      .def(py::init<const std::vector<int64_t>&, int64_t, Tensor>(), py::arg("words"), py::arg("rows"), py::arg("like"))
      .def("copy", &RowLayout::copy, py::arg("to"), py::arg("src"), py::arg("dst"), py::arg("tokens"));
  m.attr("ROW_STEPS") = (int)jla::ROW_STEPS;
}
