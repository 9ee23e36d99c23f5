// Host launchers of the serving kernels (module jax_llama_amd._C_serving): attention of a batch whose rows share prefixes,
// penalties / biases / masks on logits, and copies of cache rows. Pure HIP translation units (no torch headers).
// Every launcher returns 0 on success, <0 on a shape / argument error, >0 for a hipError_t.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace jla {

// ---- attention over shared prefixes (prefix_attn.hip)
struct PrefixAttn {
  const uint16_t *q;         // [B, S, H, 128] bf16
  const uint16_t *kp, *vp;   // prefix keys and values [G, Hkv, P, 128]; row b reads prefix b / (B / G)
  const uint16_t *ko, *vo;   // own keys and values [B, Hkv, T, 128]
  long long kp_g, kp_h, vp_g, vp_h, ko_b, ko_h, vo_b, vo_h;  // strides in elements (tokens are 128 apart)
  const int32_t* slot;       // [1]: own slot of a row's first query; null: slot0
  int slot0;
  const int32_t* prefix_len;    // optional [G]: keys of the prefix (else P)
  const int32_t* prefix_start;  // optional [G]: its first key
  const uint8_t* prefix_mask;   // optional [G, P]
  const int32_t* kv_start;      // optional [B]: first own key
  uint16_t* out;             // [B * S, H * 128] bf16
  uint16_t* out_pack;        // optional packed copy (common.h pack_off)
  float* part;               // workspace: prefix_attn_workspace floats
  int B, S, H, Hkv, G, P, T;
  int rep, n;                // query heads per kv head, rows per prefix
};
struct PrefixPlan {
  int by_row;   // column tiles of one row over prefix and own keys, else tiles over a group's rows plus each row's own keys
  int ct;       // tiles of 128 columns per (group or row, kv head)
  int ns;       // splits of their keys
  int brief;    // prefix_short_kernel; the others are not looked at but own_ct
  int own_ct;   // not by_row: tiles of 16 columns per (row, kv head)
  int own_ns;   // and splits of the own keys
  __host__ __device__ int parts() const { return ns + (by_row ? 0 : own_ns); }
};
PrefixPlan prefix_attn_plan(int B, int S, int H, int Hkv, int G, int P, int T);
long long prefix_attn_workspace(const PrefixPlan& p, int B, int S, int H);
int prefix_attn(const PrefixAttn& a, const PrefixPlan& p, hipStream_t s);

// ---- logits (logits.hip)
struct LogitsArgs {
  const float* x;            // [B, V]
  float* out;                // [B, V], or x itself
  long long ldx, ldo;        // row strides in elements
  const int32_t* history;    // optional [B, L]: token ids of each row (row stride ldh), those outside the vocabulary are ignored
  long long ldh;
  int L;
  const int32_t* length;     // [1]: places of history in use; null: length0
  int length0;
  const int32_t* start;      // optional [B]: first of them
  const uint8_t* hmask;      // optional [B, L] (row stride ldm): places that count
  long long ldm;
  int prompt_len;            // places before it are the prompt: seen, but not counted
  int vocab0;                // first token id of the columns (a vocabulary shard)
  float rep, pres, freq;     // used where the pointers are null
  const float *rep_rows, *pres_rows, *freq_rows;  // optional [B]
  const float* bias;         // optional [V], or [B, V] with row stride ldb
  long long ldb;
  const int32_t* allowed;    // optional [n_masks, ldw] bits over token ids
  long long ldw;
  int n_masks;
  const int32_t* mask_rows;  // optional [B]: row of allowed (outside [0, n_masks): everything is allowed); else row b, or 0 of one
  int B, V;
};
int process_logits(const LogitsArgs& a, hipStream_t s);

// ---- cache rows (cache_rows.hip)
struct RowSpan {             // a tensor, or several equal ones (layers) at one distance, of a cache
  uint64_t base;             // address of row 0
  long long row_bytes;       // from a row to the next
  long long layer_bytes;     // from a layer to the next
  long long run_bytes;       // from a run (a head's tokens) to the next
  long long layers, runs;    // runs: per row and layer
  long long token_bytes;     // bytes of a run per token, or 0: fixed_bytes whatever the tokens
  long long fixed_bytes;
};
// Steps (a, b) of a chain run in order, each thread at its own place of every row: b >= 0: row a (ROW_ZERO: zeros, ROW_SAVED: the saved
// one) goes to row b; b == ROW_SAVED: row a is saved. No chain writes a row that another one reads or writes.
constexpr int ROW_ZERO = -1, ROW_SAVED = -2;
constexpr int ROW_STEPS = 320, ROW_FEW = 32, ROW_SPANS = 3;  // what travels as the kernel's argument (keys, values, rows' starts)
template <int STEPS>
struct RowProgramOf {
  int32_t step[2 * STEPS];
  uint16_t chain[STEPS + 1];  // first step of each chain, and the end
  RowSpan src[ROW_SPANS], dst[ROW_SPANS];
};
using RowProgram = RowProgramOf<ROW_STEPS>;
using RowProgramFew = RowProgramOf<ROW_FEW>;
// long_program: [2 * n_steps] steps, then [n_chains + 1] first steps, on the device (programs of more than ROW_STEPS), else null.
// src, dst: the spans on the device (more than ROW_SPANS), else null. blocks: 16 KiB pieces of the span that has most
int copy_rows(const RowProgram& program, const int32_t* long_program, const RowSpan* src, const RowSpan* dst, int spans, int n_steps,
              int n_chains, int tokens, long long blocks, hipStream_t s);

}  // namespace jla
