// Copies of whole cache rows: for every tensor of a cache (or from one cache to another of the same layers), row dst[i] becomes row
// src[i], its first `tokens` tokens and all of its recurrent state, as if every source were read before anything is written.
//
// The host turns the pairs into chains of steps (bindings.cpp plan_rows); a thread walks a chain at some places (16 bytes each, or what the
// tensors' alignment allows) of every row, so that what a step reads has been overwritten by no thread but itself, and a source that
// goes to several rows is read once. Memory bounds it: each distinct source read once, each destination written once. What is written is
// not kept in the caches, nor what is read where every source goes to one row: two prompts of 517 tokens to 16 rows, 16 layers of 8
// heads, 126 -> 109 us (5.6 TB/s; with reads past the caches too 130), 24 rows of 301 tokens moved within a cache 97 -> 89 us (5.3), one
// request of 2000 tokens copied, 32 layers, 100 -> 89 us (5.9).
#include "../kernels/common.h"
#include "serving.h"

namespace jla {

constexpr int CR_THREADS = 256, CR_PLACES = 4;  // places of a thread, CR_THREADS apart: their loads are under way together

template <bool SINGLE, class T, class Step>
JLA_DEV void walk(const char* src, char* dst, long long src_row, long long dst_row, int left, Step step, int from, int to) {
  T held[CR_PLACES] = {}, saved[CR_PLACES] = {};
  int last = ROW_ZERO;
  auto read = [&](T (&t)[CR_PLACES], const char* row) {
#pragma unroll
    for (int j = 0; j < CR_PLACES; ++j)
      if (CR_THREADS * j < left) {
        const T* const at = reinterpret_cast<const T*>(row) + CR_THREADS * j;
        t[j] = SINGLE ? __builtin_nontemporal_load(at) : *at;
      }
  };
  for (int k = from; k < to; ++k) {
    const int a = step(2 * k), b = step(2 * k + 1);
    if (b == ROW_SAVED) {
      read(saved, src + a * src_row);
      continue;
    }
    if (a == ROW_SAVED || a == ROW_ZERO) {
#pragma unroll
      for (int j = 0; j < CR_PLACES; ++j) held[j] = a == ROW_SAVED ? saved[j] : T{};
    } else if (a != last) {
      read(held, src + a * src_row);
    }
    last = a;
    T* const row = reinterpret_cast<T*>(dst + b * dst_row);
#pragma unroll
    for (int j = 0; j < CR_PLACES; ++j)
      if (CR_THREADS * j < left) __builtin_nontemporal_store(held[j], row + CR_THREADS * j);
  }
}

// SINGLE: every source goes to one row (chains of one step)
template <bool LONG, bool TABLES, bool SINGLE, class Program>
__global__ void __launch_bounds__(CR_THREADS)
    copy_rows_kernel(Program program, const int32_t* __restrict__ long_program, const RowSpan* __restrict__ src_spans,
                     const RowSpan* __restrict__ dst_spans, int n_steps, int n_chains, int tokens) {
  const RowSpan s = TABLES ? src_spans[blockIdx.y] : program.src[blockIdx.y], d = TABLES ? dst_spans[blockIdx.y] : program.dst[blockIdx.y];
  const long long bytes = s.token_bytes ? s.token_bytes * tokens : s.fixed_bytes;
  if (bytes <= 0) return;
  const long long all = (long long)s.base | (long long)d.base | s.row_bytes | d.row_bytes | s.layer_bytes | d.layer_bytes | s.run_bytes | d.run_bytes | bytes;
  const int width = !(all & 15) ? 16 : !(all & 3) ? 4 : 2;
  const long long places = bytes / width;  // of a run
  const unsigned pieces = (unsigned)((places + CR_THREADS * CR_PLACES - 1) / (CR_THREADS * CR_PLACES)), runs = (unsigned)s.runs;
  auto step = [&](int i) { return LONG ? long_program[i] : program.step[i]; };
  for (unsigned long long x = blockIdx.x; x < (unsigned long long)s.layers * runs * pieces; x += gridDim.x) {
    const unsigned piece = (unsigned)(x % pieces), run = (unsigned)(x / pieces % runs), layer = (unsigned)(x / pieces / runs);
    const long long first = (long long)piece * CR_THREADS * CR_PLACES + threadIdx.x, left = places - first;
    if (left <= 0) continue;
    const int n = left < CR_THREADS * CR_PLACES ? (int)left : CR_THREADS * CR_PLACES;
    const char* const src = reinterpret_cast<const char*>(s.base) + layer * s.layer_bytes + run * s.run_bytes + first * width;
    char* const dst = reinterpret_cast<char*>(d.base) + layer * d.layer_bytes + run * d.run_bytes + first * width;
    for (int c = blockIdx.z; c < n_chains; c += gridDim.z) {
      const int from = LONG ? long_program[2 * n_steps + c] : program.chain[c];
      const int to = LONG ? long_program[2 * n_steps + c + 1] : program.chain[c + 1];
      if (width == 16) walk<SINGLE, u32x4>(src, dst, s.row_bytes, d.row_bytes, n, step, from, to);
      else if (width == 4) walk<SINGLE, uint32_t>(src, dst, s.row_bytes, d.row_bytes, n, step, from, to);
      else walk<SINGLE, uint16_t>(src, dst, s.row_bytes, d.row_bytes, n, step, from, to);
    }
  }
}

// (the arguments lie in the host's memory: most calls take a few steps and should not carry 4 KiB)
template <bool LONG, bool TABLES, class Program>
static void launch(dim3 grid, hipStream_t s, const Program& program, const int32_t* long_program, const RowSpan* src, const RowSpan* dst, int n_steps,
                   int n_chains, int tokens) {
  if (n_steps == n_chains)
    copy_rows_kernel<LONG, TABLES, true><<<grid, CR_THREADS, 0, s>>>(program, long_program, src, dst, n_steps, n_chains, tokens);
  else
    copy_rows_kernel<LONG, TABLES, false><<<grid, CR_THREADS, 0, s>>>(program, long_program, src, dst, n_steps, n_chains, tokens);
}

int copy_rows(const RowProgram& program, const int32_t* long_program, const RowSpan* src, const RowSpan* dst, int spans, int n_steps,
              int n_chains, int tokens, long long blocks, hipStream_t s) {
  if (spans <= 0 || n_chains <= 0 || blocks <= 0) return 0;
  if (spans > 65535 || tokens < 0 || (!src && spans > ROW_SPANS) || !src != !dst || (!long_program && n_steps > ROW_STEPS)) return -1;
  const dim3 grid((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20), spans, n_chains < 4096 ? n_chains : 4096);
  if (long_program || n_steps <= ROW_FEW) {
    RowProgramFew few{};
    if (!long_program) {
      for (int i = 0; i < 2 * n_steps; ++i) few.step[i] = program.step[i];
      for (int i = 0; i <= n_chains; ++i) few.chain[i] = program.chain[i];
    }
    if (!src)
      for (int i = 0; i < spans; ++i) few.src[i] = program.src[i], few.dst[i] = program.dst[i];
    if (long_program && src) launch<true, true>(grid, s, few, long_program, src, dst, n_steps, n_chains, tokens);
    else if (long_program) launch<true, false>(grid, s, few, long_program, src, dst, n_steps, n_chains, tokens);
    else if (src) launch<false, true>(grid, s, few, long_program, src, dst, n_steps, n_chains, tokens);
    else launch<false, false>(grid, s, few, long_program, src, dst, n_steps, n_chains, tokens);
  } else if (src) {
    launch<false, true>(grid, s, program, long_program, src, dst, n_steps, n_chains, tokens);
  } else {
    launch<false, false>(grid, s, program, long_program, src, dst, n_steps, n_chains, tokens);
  }
  JLA_CHECK_LAUNCH();
  return 0;
}

}  // namespace jla
