// Copies of whole cache rows: for every tensor of a cache (or from one cache to another of the same layers), row dst[i] becomes row
// src[i], its first `tokens` tokens and all of its recurrent state, as if every source were read before anything is written.
//
// The host turns the pairs into chains of steps (ops/cache_rows.py); a thread walks a chain at one place (16 bytes, or what the
// tensors' alignment allows) of every row, so that what a step reads has been overwritten by no thread but itself, and a source that
// goes to several rows is read once. Memory bounds it: each distinct source read once, each destination written once.
#include "../kernels/common.h"
#include "serving.h"

namespace jla {

constexpr int CR_THREADS = 256;

template <class T, class Step>
JLA_DEV void walk(const RowSpan& s, const RowSpan& d, long long run, long long places, Step step, int from, int to) {
  for (long long i = (long long)blockIdx.x * CR_THREADS + threadIdx.x; i < places; i += (long long)gridDim.x * CR_THREADS) {
    const long long r = i / run, at = (i - r * run) * (long long)sizeof(T);
    const char* const src = reinterpret_cast<const char*>(s.base) + r * s.run_bytes + at;
    char* const dst = reinterpret_cast<char*>(d.base) + r * d.run_bytes + at;
    T held{}, saved{};
    int last = ROW_ZERO;
    for (int k = from; k < to; ++k) {
      const int a = step(2 * k), b = step(2 * k + 1);
      if (b == ROW_SAVED) {
        saved = *reinterpret_cast<const T*>(src + a * s.row_bytes);
        continue;
      }
      if (a == ROW_SAVED) held = saved;
      else if (a == ROW_ZERO) held = T{};
      else if (a != last) held = *reinterpret_cast<const T*>(src + a * s.row_bytes);
      last = a;
      *reinterpret_cast<T*>(dst + b * d.row_bytes) = held;
    }
  }
}

template <bool LONG>
__global__ void __launch_bounds__(CR_THREADS)
    copy_rows_kernel(const RowSpan* __restrict__ src, const RowSpan* __restrict__ dst, RowProgram program, const int32_t* __restrict__ long_program,
                     int n_steps, int n_chains, int tokens) {
  const RowSpan s = src[blockIdx.y], d = dst[blockIdx.y];
  const long long bytes = s.token_bytes ? (long long)s.token_bytes * tokens : s.fixed_bytes;
  if (bytes <= 0) return;
  const long long shape = (long long)s.base | (long long)d.base | s.row_bytes | d.row_bytes | s.run_bytes | d.run_bytes | bytes;
  auto step = [&](int i) { return LONG ? long_program[i] : program.step[i]; };
  for (int c = blockIdx.z; c < n_chains; c += gridDim.z) {
    const int from = LONG ? long_program[2 * n_steps + c] : program.chain[c];
    const int to = LONG ? long_program[2 * n_steps + c + 1] : program.chain[c + 1];
    if (!(shape & 15)) walk<u32x4>(s, d, bytes / 16, bytes / 16 * s.runs, step, from, to);
    else if (!(shape & 3)) walk<uint32_t>(s, d, bytes / 4, bytes / 4 * s.runs, step, from, to);
    else walk<uint16_t>(s, d, bytes / 2, bytes / 2 * s.runs, step, from, to);
  }
}

// widest: bytes of a row in the largest tensor
int copy_rows(const RowSpan* src, const RowSpan* dst, int spans, const RowProgram& program, const int32_t* long_program, int n_steps,
              int n_chains, int tokens, long long widest, hipStream_t s) {
  if (spans <= 0 || n_chains <= 0 || widest <= 0) return 0;
  if (spans > 65535 || tokens < 0) return -1;
  long long x = (widest / 16 + CR_THREADS - 1) / CR_THREADS;
  if (x < 1) x = 1;
  if (x > 4096) x = 4096;
  const dim3 grid((int)x, spans, n_chains < 4096 ? n_chains : 4096);
  if (long_program) copy_rows_kernel<true><<<grid, CR_THREADS, 0, s>>>(src, dst, program, long_program, n_steps, n_chains, tokens);
  else copy_rows_kernel<false><<<grid, CR_THREADS, 0, s>>>(src, dst, program, long_program, n_steps, n_chains, tokens);
  JLA_CHECK_LAUNCH();
  return 0;
}

}  // namespace jla
