// Penalties for repeated tokens, biases and masks on logits. Of token v of row b, over the row's history (place i of [start[b], length),
// where hmask is set):
//   count = places from prompt_len on that hold v, seen = some place holds v
//   x <- seen ? (x < 0 ? x r : x / r) : x;   x <- x - f count - (count > 0 ? p : 0);   x <- x + bias;   x <- allowed ? x : -inf.
//
// A workgroup takes LG_CHUNK columns of a row and counts the history's tokens among them in LDS (integers: the order of the atomics
// does not show), so nothing about a row is kept between calls and a captured step needs the token buffer and its length alone.
#include "../kernels/common.h"
#include "serving.h"

namespace jla {

constexpr int LG_CHUNK = 8192, LG_THREADS = 256;
constexpr uint32_t LG_PROMPT = 0x80000000u;  // in the prompt; below: the count

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // (rows of odd length)

struct Penalties {
  float r, p, f;
  JLA_DEV float operator()(float x, uint32_t seen) const {
    if (!seen) return x;
    const uint32_t count = seen & ~LG_PROMPT;
    x = x < 0.f ? x * r : x / r;
    return x - f * (float)count - (count ? p : 0.f);
  }
};

// fn(column within the chunk, place) for the places of the row's history in this chunk
template <class F>
JLA_DEV void for_history(const LogitsArgs& a, int row, int c0, int n, F fn) {
  const int to = min(a.length[0], a.L);
  const int32_t* h = a.history + row * a.ldh;
  const uint8_t* m = a.hmask ? a.hmask + row * a.ldm : nullptr;
  for (int i = max(a.start ? a.start[row] : 0, 0) + (int)threadIdx.x; i < to; i += LG_THREADS) {
    const unsigned t = (unsigned)h[i] - (unsigned)a.vocab0 - (unsigned)c0;
    if (t < (unsigned)n && (!m || m[i])) fn(t, i);
  }
}

// DENSE: every column goes from x to out. Else out is x and only seen columns change.
template <bool DENSE, bool HISTORY>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(LogitsArgs a, int row0) {
  __shared__ __attribute__((aligned(16))) uint32_t seen[HISTORY ? LG_CHUNK : 4];
  const int row = row0 + blockIdx.y, c0 = blockIdx.x * LG_CHUNK, n = min(LG_CHUNK, a.V - c0);
  const float* x = a.x + row * a.ldx + c0;
  float* out = a.out + row * a.ldo + c0;
  Penalties pen{1.f, 0.f, 0.f};
  if constexpr (HISTORY) {
    pen.r = a.rep_rows ? a.rep_rows[row] : a.rep;
    pen.p = a.pres_rows ? a.pres_rows[row] : a.pres;
    pen.f = a.freq_rows ? a.freq_rows[row] : a.freq;
    for (int i = 4 * threadIdx.x; i < LG_CHUNK; i += 4 * LG_THREADS) *reinterpret_cast<u32x4*>(seen + i) = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    for_history(a, row, c0, n, [&](unsigned t, int i) {
      if (i >= a.prompt_len) atomicAdd(&seen[t], 1u);
      else atomicOr(&seen[t], LG_PROMPT);
    });
    __syncthreads();
    if constexpr (!DENSE) {
      for_history(a, row, c0, n, [&](unsigned t, int) {
        const uint32_t s = atomicExch(&seen[t], 0u);  // the first place to come takes the token
        if (s) out[t] = pen(out[t], s);
      });
      return;
    }
  }
  const float* bias = a.bias ? a.bias + row * a.ldb + c0 : nullptr;
  const uint32_t* words = nullptr;
  if (a.allowed) {
    const int r = a.mask_rows ? a.mask_rows[row] : (a.n_masks == 1 ? 0 : row);
    if (r >= 0 && r < a.n_masks) words = reinterpret_cast<const uint32_t*>(a.allowed) + r * a.ldw;
  }
  auto one = [&](int v, float f) {
    if constexpr (HISTORY) f = pen(f, seen[v]);
    if (bias) f += bias[v];
    if (words) {
      const int t = a.vocab0 + c0 + v;
      if (!(words[t >> 5] >> (t & 31) & 1)) f = -INFINITY;  // (whatever stood there, a NaN too)
    }
    return f;
  };
  for (int v = 4 * threadIdx.x; v < n; v += 4 * LG_THREADS) {
    if (v + 4 <= n) {
      f32x4 f = *reinterpret_cast<const f32x4u*>(x + v);
      if constexpr (HISTORY) {
        const u32x4 s = *reinterpret_cast<const u32x4*>(seen + v);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = pen(f[e], s[e]);
      }
      if (bias) f += *reinterpret_cast<const f32x4u*>(bias + v);
      if (words) {
        const int t = a.vocab0 + c0 + v, sh = t & 31;
        uint32_t bits = words[t >> 5] >> sh;
        if (sh > 28) bits |= words[(t >> 5) + 1] << (32 - sh);  // (column v + 3 is in that word)
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = bits >> e & 1 ? f[e] : -INFINITY;
      }
      *reinterpret_cast<f32x4u*>(out + v) = f;
    } else {
      for (int e = v; e < n; ++e) out[e] = one(e, x[e]);
    }
  }
}

int process_logits(const LogitsArgs& a, hipStream_t s) {
  if (a.B <= 0 || a.V <= 0) return 0;
  if (a.history && !a.length) return -1;
  const bool dense = a.bias || a.allowed || a.out != a.x;
  if (!dense && !a.history) return 0;
  for (int r0 = 0; r0 < a.B; r0 += 65535) {  // (the grid's second axis)
    const dim3 grid((a.V + LG_CHUNK - 1) / LG_CHUNK, a.B - r0 < 65535 ? a.B - r0 : 65535);
    if (!dense) logits_kernel<false, true><<<grid, LG_THREADS, 0, s>>>(a, r0);
    else if (a.history) logits_kernel<true, true><<<grid, LG_THREADS, 0, s>>>(a, r0);
    else logits_kernel<true, false><<<grid, LG_THREADS, 0, s>>>(a, r0);
    JLA_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace jla
