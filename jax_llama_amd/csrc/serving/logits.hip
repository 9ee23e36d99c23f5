// Penalties for repeated tokens, biases and masks on logits. Of token v of row b, over the row's history (place i of [start[b], length),
// where hmask is set):
//   count = places from prompt_len on that hold v, seen = some place holds v
//   x <- seen ? (x < 0 ? x r : x / r) : x;   x <- x - f count - (count > 0 ? p : 0);   x <- x + bias;   x <- allowed ? x : -inf.
//
// A workgroup takes 1024 GROUPS columns of a row and counts the history's tokens among them in LDS (integers: the order of the atomics
// does not show), so nothing about a row is kept between calls and a captured step needs the token buffer and its length alone.
//
// Memory bounds it: logits read and written once. The logits of a workgroup are on their way to registers while it looks through the
// history (1024 rows of 128256, 384 places: 260 us with the loads behind it, 213 before). Of 8192 columns a workgroup few of them fit a
// compute unit and their reads, counts and writes come in step (213 us, 64 rows with masks and 2048 places 18.3), of 4096 they spread out
// (200 us, 5.2 TB/s; 16.4), of 2048 and 1024 the history is looked through too often (199, 224 us; 18.5, 19.7). Few rows take
// 1024 columns, for more workgroups: 1 x 32000 5.0 -> 4.0 us.
#include "../kernels/common.h"
#include "serving.h"

namespace jla {

constexpr int LG_THREADS = 256;
constexpr uint32_t LG_PROMPT = 0x80000000u;  // in the prompt; below: the count

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // (rows of odd length)
typedef int i32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct Penalties {
  float r, p, f;
  JLA_DEV float operator()(float x, uint32_t seen) const {
    if (!seen) return x;
    const uint32_t count = seen & ~LG_PROMPT;
    x = x < 0.f ? x * r : x / r;
    return x - f * (float)count - (count ? p : 0.f);
  }
};

// fn(column within the chunk, place) for the places of the row's history in this chunk, eight of them under way per thread. Places are
// unsigned: `to` is below 2^31, so that a thread's next place past it does not wrap.
template <class F>
JLA_DEV void for_history(const LogitsArgs& a, int row, int c0, int n, F fn) {
  const unsigned to = (unsigned)max(min(a.length ? a.length[0] : a.length0, a.L), 0);
  const int32_t* h = a.history + row * a.ldh;
  const uint8_t* m = a.hmask ? a.hmask + row * a.ldm : nullptr;
  const unsigned lowest = (unsigned)a.vocab0 + (unsigned)c0;
  for (unsigned i = min((unsigned)max(a.start ? a.start[row] : 0, 0), to) + 4 * threadIdx.x; i < to; i += 8 * LG_THREADS) {
    unsigned t[2][4];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const unsigned at = i + 4 * LG_THREADS * g;
      if (at + 4 <= to) {
        const i32x4u v = *reinterpret_cast<const i32x4u*>(h + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[g][e] = (unsigned)v[e] - lowest;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[g][e] = at + e < to ? (unsigned)h[at + e] - lowest : ~0u;
      }
    }
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned at = i + 4 * LG_THREADS * g + e;
        if (t[g][e] < (unsigned)n && (!m || m[at])) fn(t[g][e], (int)at);
      }
  }
}

// DENSE: every column goes from x to out, a thread's in GROUPS accesses, all under way before the history is looked through. Else out is x
// and only seen columns change.
template <bool DENSE, bool HISTORY, int GROUPS>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(LogitsArgs a, int row0) {
  constexpr int LG_CHUNK = 4 * LG_THREADS * GROUPS;
  __shared__ __attribute__((aligned(16))) uint32_t seen[HISTORY ? LG_CHUNK : 4];
  const int row = row0 + blockIdx.y, c0 = blockIdx.x * LG_CHUNK, n = min(LG_CHUNK, a.V - c0);
  const float* x = a.x + row * a.ldx + c0;
  float* out = a.out + row * a.ldo + c0;
  const int first = 4 * threadIdx.x;
  f32x4 f[GROUPS];
  if constexpr (DENSE) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int v = first + 4 * LG_THREADS * g;
      if (v + 4 <= n) f[g] = *reinterpret_cast<const f32x4u*>(x + v);
    }
  }
  Penalties pen{1.f, 0.f, 0.f};
  if constexpr (HISTORY) {
    pen.r = a.rep_rows ? a.rep_rows[row] : a.rep;
    pen.p = a.pres_rows ? a.pres_rows[row] : a.pres;
    pen.f = a.freq_rows ? a.freq_rows[row] : a.freq;
    for (int i = first; i < n; i += 4 * LG_THREADS) *reinterpret_cast<u32x4*>(seen + i) = u32x4{0u, 0u, 0u, 0u};
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
    }
  }
  if constexpr (DENSE) {
    const float* bias = a.bias ? a.bias + row * a.ldb + c0 : nullptr;
    const uint32_t* words = nullptr;
    if (a.allowed) {
      const int r = a.mask_rows ? a.mask_rows[row] : (a.n_masks == 1 ? 0 : row);
      if (r >= 0 && r < a.n_masks) words = reinterpret_cast<const uint32_t*>(a.allowed) + r * a.ldw;
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int v = first + 4 * LG_THREADS * g;
      if (v + 4 <= n) {
        if constexpr (HISTORY) {
          const u32x4 s = *reinterpret_cast<const u32x4*>(seen + v);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[g][e] = pen(f[g][e], s[e]);
        }
        if (bias) f[g] += *reinterpret_cast<const f32x4u*>(bias + v);
        if (words) {
          const int t = a.vocab0 + c0 + v, sh = t & 31;
          uint32_t bits = words[t >> 5] >> sh;
          if (sh > 28) bits |= words[(t >> 5) + 1] << (32 - sh);  // (column v + 3 is in that word)
#pragma unroll
          for (int e = 0; e < 4; ++e) f[g][e] = bits >> e & 1 ? f[g][e] : -INFINITY;  // (whatever stood there, a NaN too)
        }
        *reinterpret_cast<f32x4u*>(out + v) = f[g];
      } else {
        for (int e = v; e < n; ++e) {  // (a row's last three columns at most)
          float o = x[e];
          if constexpr (HISTORY) o = pen(o, seen[e]);
          if (bias) o += bias[e];
          const int t = a.vocab0 + c0 + e;
          if (words && !(words[t >> 5] >> (t & 31) & 1)) o = -INFINITY;
          out[e] = o;
        }
      }
    }
  }
}

template <int GROUPS>
static int launch(const LogitsArgs& a, bool dense, hipStream_t s) {
  const int chunks = (a.V + 4 * LG_THREADS * GROUPS - 1) / (4 * LG_THREADS * GROUPS);
  for (int r0 = 0; r0 < a.B; r0 += 65535) {  // (the grid's second axis)
    const dim3 grid(chunks, a.B - r0 < 65535 ? a.B - r0 : 65535);
    if (!dense) logits_kernel<false, true, GROUPS><<<grid, LG_THREADS, 0, s>>>(a, r0);
    else if (a.history) logits_kernel<true, true, GROUPS><<<grid, LG_THREADS, 0, s>>>(a, r0);
    else logits_kernel<true, false, GROUPS><<<grid, LG_THREADS, 0, s>>>(a, r0);
    JLA_CHECK_LAUNCH();
  }
  return 0;
}

int process_logits(const LogitsArgs& a, hipStream_t s) {
  if (a.B <= 0 || a.V <= 0) return 0;
  bool dense = a.bias || a.allowed || a.out != a.x;
  if (!dense && !a.history) return 0;
  // In place, penalties alone change the history's tokens, each somewhere else in memory: less than all columns up to a place in 40 or so
  // (1024 rows of 128256, us in place | every column: 384 places 58 | 192, 4096 286 | 190; 64 rows 5.8 | 11.0, 16.4 | 14.7).
  dense = dense || a.L > a.V / 40;
  const long long groups = (long long)a.B * ((a.V + 4095) / 4096);
  return groups <= 512 ? launch<1>(a, dense, s) : launch<4>(a, dense, s);  // (16 rows of 128256: 10.3, 11.0 us)
}

}  // namespace jla
