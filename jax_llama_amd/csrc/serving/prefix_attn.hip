// Attention of a batch whose rows share prefixes: query (b, s) of head h attends the keys of prefix g = b / (B / G) that lie in
// [prefix_start[g], prefix_len[g]) (and are set in prefix_mask) and its row's own keys in [kv_start[b], slot + s]:
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = q . k_j log2(e) / sqrt(128),   m = max_j x_j.
// A query without keys gives zeros.
//
// The keys of a set are taken in parts; a part leaves (m, l, O) = (its maximum, sum of 2^(x - m), sum of 2^(x - m) v) in 32 bits, and
// the parts of a query join as m' = max m_i, l' = sum l_i 2^(m_i - m'), O' = sum O_i 2^(m_i - m').
//
// Columns. The queries of one kv head that read the same keys are the columns of S^T = K Q^T: for a prefix n S rep of them (n rows of
// its group, rep query heads per kv head, column c = token (c / rep), head (c % rep)), for a row's own keys S rep. So a prefix is
// read once per 128 columns instead of once per row.
#include <atomic>
#include <type_traits>

#include "../kernels/common.h"
#include "serving.h"

namespace jla {

constexpr int PA_DH = 128;
constexpr int PA_KT = 64;                         // keys per tile of a workgroup's 128 columns
constexpr int PA_TILE = PA_KT * PA_DH * 2;        // 16 KiB
constexpr int PA_STEP = 32;                       // keys per step of a wave's 16 columns
constexpr int PA_COLS = 128;

// A step's 32 products in their order: 0 .. 15 of keys (two blocks of 32, 16 dims each), 16 + 4 ks + dt of values
constexpr int PA_AHEAD = 3;  // operands are read from LDS this many products ahead (the first ones of keys: see the clearing of values)
constexpr int PA_ORDER[32] = {0, 1, 2, 16, 3, 17, 4, 18, 5, 19, 6, 7, 8, 20, 9, 21, 10, 22, 11, 23, 12, 13, 24, 14, 25, 15, 26, 27, 28, 29, 30, 31};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// byte offset of 16-byte chunk ch (0..15) of row `row` of a [rows][128 bf16] image in LDS: neither ds_read_b128 of rows nor
// ds_read_b64_tr_b16 of columns meets a bank twice
JLA_DEV int pa_off(int row, int ch) { return 256 * row + 16 * (ch ^ (((row & 3) << 2) | ((row >> 2) & 3))); }

JLA_DEV f32x16 mfma32(const u32x4 a, const u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
JLA_DEV u32x2 ld_tr(const char* lds, int off) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + off)));
}

// LDS-DMA of 16 bytes a lane from base + off[j] to LDS bytes lds_wave + 4096 j .. + 1023 of a wave (kernels/common.h glds16_asm)
JLA_DEV void glds16x4(const void* base, const int (&off)[4], unsigned lds_wave) {
  asm volatile(
      "s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %4\n\t"
      "s_add_i32 m0, m0, 4096\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %4\n\t"
      "s_add_i32 m0, m0, 4096\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %4\n\t"
      "s_add_i32 m0, m0, 4096\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %4" ::"v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "s"(lds_wave)
      : "memory", "m0", "scc");
}

JLA_DEV int own_slot(const PrefixAttn& a) { return a.slot ? a.slot[0] : a.slot0; }

// keys [lo, hi) of one sequence in tiles aligned to its start
struct KeyRange {
  const bf16_t *k, *v;
  int lo, hi, limit;  // limit: rows that may be read
  const uint8_t* mask;
  JLA_DEV int first(int tile) const { return lo / tile * tile; }
  JLA_DEV int tiles(int tile) const { return lo < hi ? (hi - 1) / tile - lo / tile + 1 : 0; }
};

JLA_DEV KeyRange prefix_keys(const PrefixAttn& a, int g, int kvh) {
  KeyRange r;
  r.k = a.kp + g * a.kp_g + kvh * a.kp_h;
  r.v = a.vp + g * a.vp_g + kvh * a.vp_h;
  r.lo = a.prefix_start ? max(a.prefix_start[g], 0) : 0;
  r.hi = a.prefix_len ? min(a.prefix_len[g], a.P) : a.P;
  r.limit = a.P;
  r.mask = a.prefix_mask ? a.prefix_mask + (size_t)g * a.P : nullptr;
  return r;
}
// up to the slot of query s_last
JLA_DEV KeyRange own_keys(const PrefixAttn& a, int b, int kvh, int s_last) {
  KeyRange r;
  r.k = a.ko + b * a.ko_b + kvh * a.ko_h;
  r.v = a.vo + b * a.vo_b + kvh * a.vo_h;
  r.lo = a.kv_start ? max(a.kv_start[b], 0) : 0;
  r.hi = min(own_slot(a) + s_last + 1, a.T);
  r.limit = a.T;
  r.mask = nullptr;
  return r;
}

// A part's share of the workspace: [parts][queries][128] sums, then [parts][queries][2] (maximum, sum of weights)
JLA_DEV float* part_sums(const PrefixAttn& a, int part, size_t qh) { return a.part + ((size_t)part * a.B * a.S * a.H + qh) * PA_DH; }
JLA_DEV float* part_stats(const PrefixAttn& a, int parts, int part, size_t qh) {
  const size_t n = (size_t)a.B * a.S * a.H;
  return a.part + n * PA_DH * parts + (part * n + qh) * 2;
}
JLA_DEV u32x2 result4(const float* o, float inv) { return u32x2{pack2bf(o[0] * inv, o[1] * inv), pack2bf(o[2] * inv, o[3] * inv)}; }

// ---- 128 columns of a workgroup of four waves, 32 a wave (a lane's column is lane & 31). Tiles of 64 keys go to LDS by LDS-DMA, two
// slots each for keys and values; S^T = K Q^T leaves a column's scores in its two lanes, which are the operand of O^T += V^T P^T as
// they are (V^T by transposing reads). 64 columns a wave would halve the reads of LDS, but leave one wave a SIMD, which issues too few
// instructions (330 us where this takes 255). 16 rows of 200 queries behind 4096 keys 225 us (979 TFLOP/s; the library's large product reaches
// 1360), 64 rows behind 65536 keys 91 us with the join (0.74 PFLOP/s, 3.1 TB/s).
JLA_DEV void column_tile(const PrefixAttn& a, const PrefixPlan& p, int part, int kvh, size_t tok0, int ncols, int ct, const KeyRange& pre,
                         const KeyRange& own, char* lds) {
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, col = lane & 31, rep = a.rep;
  const int c0 = (4 * ct + w) * 32;
  const bool active = c0 < ncols;  // (the wave's; the others help to stage)
  const float scale = 1.4426950408889634f / 11.313708498984761f;
  // a column's slot; those of the wave's first and last columns
  const int slot = own_slot(a), at_first = slot + min(c0, ncols - 1) / rep, at_last = slot + min(c0 + 31, ncols - 1) / rep;
  const int c = min(c0 + col, ncols - 1), at = slot + c / rep;
  const size_t qh = (tok0 + c / rep) * a.H + kvh * rep + c % rep;
  u32x4 qf[8];
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) qf[ks] = *reinterpret_cast<const u32x4*>(a.q + qh * PA_DH + 16 * ks + 8 * hi);
  f32x16 o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  float m_run = -INFINITY, m_use = 0.f, l_run = 0.f, sum = 0.f;
  u32x4 pf = {0u, 0u, 0u, 0u};

  const int n_pre = pre.tiles(PA_KT), n_all = n_pre + own.tiles(PA_KT);
  const int from = (int)((long long)n_all * part / p.ns), to = (int)((long long)n_all * (part + 1) / p.ns);
  const int gq = (lane & 15) >> 2, gp = lane & 3, G = lane >> 4;
  struct Tile {
    const bf16_t *k, *v;
    const uint8_t* mask;
    int t0, lo, hi, limit;
    bool own;
  };
  auto tile_of = [&](int i) {
    return i < n_pre ? Tile{pre.k, pre.v, pre.mask, pre.first(PA_KT) + i * PA_KT, pre.lo, pre.hi, pre.limit, false}
                     : Tile{own.k, own.v, nullptr, own.first(PA_KT) + (i - n_pre) * PA_KT, own.lo, own.hi, own.limit, true};
  };
  // a bit for each of a tile's keys that the range and the mask leave (all lanes)
  auto kept_of = [&](const Tile& t) -> uint64_t {
    if (t.t0 >= t.lo && t.t0 + PA_KT <= t.hi && !t.mask) return ~0ull;
    const int key = t.t0 + lane;
    return __ballot(key >= t.lo && key < t.hi && (!t.mask || t.mask[min(key, t.limit - 1)]));
  };
  // A wave issues an instruction every 8 to 10 cycles, scalar ones too, and that bounds a step: what most tiles need is kept few. Tiles
  // [plain, plain + n_plain) are the prefix's, whole and without a mask; from `past` on nothing is this wave's.
  const int plain = pre.lo % PA_KT ? 1 : 0, n_plain = pre.mask ? 0 : max(0, n_pre - plain - (pre.hi % PA_KT ? 1 : 0));
  auto is_plain = [&](int i) { return (unsigned)(i - plain) < (unsigned)n_plain; };
  const int past = !active ? 0 : min(to, n_pre + max(0, ((at_last - own.first(PA_KT)) >> 6) + 1));
  auto slot_k = [&](int par) { return lds + par * PA_TILE; };
  auto slot_v = [&](int par) { return lds + (2 + par) * PA_TILE; };
  const unsigned lds_w = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds + 1024 * w;
  // 1-KiB blocks of 4 rows, lane L fills row L / 16, place L % 16 of its block (by asm: for the builtin the compiler waits before the
  // next read of LDS)
  int off[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) off[j] = 256 * (4 * (w + 4 * j) + (lane >> 4)) + 16 * ((lane & 15) ^ (((lane >> 4) << 2) | w));
  auto stage = [&](const bf16_t* plain_at, const bf16_t* pre_at, const bf16_t* own_at, int i, int to_slot) {
    if (is_plain(i)) {
      glds16x4(plain_at + (size_t)i * (PA_KT * PA_DH), off, lds_w + to_slot * PA_TILE);
    } else {
      const Tile t = tile_of(i);
      int at_row[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) at_row[j] = off[j] - 256 * max(0, 4 * (w + 4 * j) + (lane >> 4) - (t.limit - 1 - t.t0));
      glds16x4((t.own ? own_at : pre_at) + (size_t)t.t0 * PA_DH, at_row, lds_w + to_slot * PA_TILE);
    }
  };
  const size_t skipped = (size_t)pre.first(PA_KT) * PA_DH;
  auto stage_k = [&](int i, int par) { stage(pre.k + skipped, pre.k, own.k, i, par); };
  auto stage_v = [&](int i, int par) { stage(pre.v + skipped, pre.v, own.v, i, 2 + par); };
  // Tile i: K(i + 1) and V(i) are there, K(i + 2) and V(i + 1) on their way to the slots that tile i - 1 is done with. The scores of
  // tile i + 1 stand among the PV products of tile i, the exponentials of a key step among the products of the one before: the matrix
  // unit (1024 cycles a tile and wave) and the vector unit (about 700) work side by side. 16 rows of 200 queries behind 4096 keys, us: the
  // products in this order with their operands PA_AHEAD before them 246 (the compiler's, each operand read just before its product, 255),
  // the maximum as one chain 234, the products before another wave's vector work 225.
  f32x16 sa[2], sb[2];
  const int k_off = pa_off(col, hi), v_off = pa_off(4 * (G >> 1) + gq, 2 * (G & 1) + (gp >> 1)) + 8 * (gp & 1);
  auto key_frag = [&](const char* kt, int f) { return *reinterpret_cast<const u32x4*>(kt + (k_off ^ (32 * (f >> 1))) + 8192 * (f & 1)); };
  auto score = [&](f32x16 (&s)[2], const u32x4 k, int f) { s[f & 1] = mfma32(k, qf[f >> 1], s[f & 1]); };
  auto clear = [&](f32x16 (&s)[2]) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[0][e] = s[1][e] = 0.f;
  };
  auto largest = [&](const f32x16 (&s)[2]) {
    float m = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) m = fmaxf(m, s[kb][e]);
    return m;
  };
  // weights of key step ks, in bf16 for the matrix cores (half a step, 2^-8, at most; their sum is of the unrounded ones)
  auto weights = [&](const f32x16 (&s)[2], int ks) {
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = __builtin_amdgcn_exp2f(fmaf(s[ks >> 1][8 * (ks & 1) + j], scale, -m_use));
      sum += e[j];
    }
    return pack8(e);
  };
  // what a tile needs before its PV: masks, the running maximum (it moves, and the sums with it, only where it grew by more than 8:
  // 2^(x - m) stays below 256), the weights of its first key step. raw: the largest score before masks
  auto enter = [&](int i, uint64_t kept, f32x16 (&s)[2], float raw) {
    const Tile t = tile_of(i);
    if (!is_plain(i) && (kept != ~0ull || (t.own && t.t0 + PA_KT - 1 > at_first))) {
      uint64_t ok = kept;  // element e of block kb is key t0 + 4 hi + 32 kb + (e & 3) + 8 (e >> 2)
      const int n = at - t.t0 + 1;
      if (t.own && n < PA_KT) ok = n > 0 ? ok & ~(~0ull << n) : 0ull;
      ok >>= 4 * hi;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t all = __builtin_amdgcn_sbfe((uint32_t)(ok >> (32 * kb)), (e & 3) + 8 * (e >> 2), 1);
          s[kb][e] = __uint_as_float((__float_as_uint(s[kb][e]) & all) | (0xff800000u & ~all));
        }
      raw = largest(s);
    }
    const float most = lane_max32(raw) * scale;
    if (__ballot(most > m_run + 8.f)) {
      const float m_new = fmaxf(m_run, most);
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
      l_run *= alpha;
      m_run = m_new;
      m_use = m_new == -INFINITY ? 0.f : m_new;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
    }
    sum = 0.f;
    pf = weights(s, 0);
  };
  auto value_frag = [&](const char* vt, int ks, int dt) {
    const u32x2 lo4 = ld_tr(vt, (v_off ^ (64 * dt)) + 4096 * ks), hi4 = ld_tr(vt, (v_off ^ (64 * dt) ^ 32) + 2048 + 4096 * ks);
    return u32x4{lo4[0], lo4[1], hi4[0], hi4[1]};
  };
  uint64_t kept = ~0ull;  // tile i's
  auto step = [&](int i, auto parity, f32x16 (&s)[2], f32x16 (&next)[2]) {
    constexpr int par = decltype(parity)::value;
    auto fetch = [&](int n) {
      const int f = PA_ORDER[n];
      return f < 16 ? key_frag(slot_k(par ^ 1), f) : value_frag(slot_v(par), (f - 16) >> 2, (f - 16) & 3);
    };
    u32x4 fr[PA_AHEAD + 1];
#pragma unroll
    for (int n = 0; n < PA_AHEAD; ++n) fr[n] = fetch(n);
    const uint64_t kept_next = is_plain(i + 1) || i + 1 >= to ? ~0ull : kept_of(tile_of(i + 1));
    if (i + 2 < to) stage_k(i + 2, par);
    if (i + 1 < to) stage_v(i + 1, par ^ 1);
    if (kept != ~0ull) {  // values of keys that nobody attends may be anything: 0 x NaN would not be 0
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = (tid >> 4) + 16 * j;
        if (!(kept >> row & 1)) *reinterpret_cast<u32x4*>(slot_v(par) + 256 * row + 16 * (tid & 15)) = u32x4{0u, 0u, 0u, 0u};
      }
      __syncthreads();
    }
    if (i < past) {
      __builtin_amdgcn_s_setprio(1);
      clear(next);
      float e[8], most0 = -INFINITY, most1 = -INFINITY;
      // (what an empty asm reads is computed before it: products and weights have no other order among themselves)
      u32x4 after = pf;
#pragma unroll
      for (int n = 0; n < 32; ++n) {
        if (n + PA_AHEAD < 32) fr[(n + PA_AHEAD) % (PA_AHEAD + 1)] = fetch(n + PA_AHEAD);
        // the weights of the next key step: an element a product, its sum one later, their packing before the step ends
        const int ks = n < 20 ? n / 10 : n < 28 ? 2 : 3, q = n < 20 ? n % 10 : (n - 20) % 8;
        if (ks < 3) {
          const int first = ks == 2 ? (q ? q + 1 : 0) : q, count = ks == 2 ? (q == 0 ? 2 : q < 7 ? 1 : 0) : q < 8 ? 1 : 0;
#pragma unroll
          for (int j = first; j < first + count; ++j) {
            e[j] = __builtin_amdgcn_exp2f(fmaf(s[(ks + 1) >> 1][8 * ((ks + 1) & 1) + j], scale, -m_use));
            asm volatile("" ::"v"(e[j]));
            if (j) {
              sum += e[j - 1];
              asm volatile("" ::"v"(sum));
            }
          }
          if (q == (ks == 2 ? 7 : 8)) {
            sum += e[7];
            after = pack8(e);
          }
        } else {  // the largest of the next tile's scores
#pragma unroll
          for (int j = 4 * q; j < 4 * q + 4; j += 2) {
            most0 = fmaxf(fmaxf(most0, next[0][j]), next[0][j + 1]);
            most1 = fmaxf(fmaxf(most1, next[1][j]), next[1][j + 1]);
          }
        }
        const int f = PA_ORDER[n];
        if (f < 16) {
          score(next, fr[n % (PA_AHEAD + 1)], f);
          asm volatile("" ::"v"(next[f & 1]));
        } else {
          o[f & 3] = mfma32(fr[n % (PA_AHEAD + 1)], pf, o[f & 3]);
          asm volatile("" ::"v"(o[f & 3]));
        }
        if (n == 9 || n == 19 || n == 27) pf = after;
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      l_run += sum;  // (this half's keys; the halves meet at the end)
      float raw = fmaxf(most0, most1);
      asm volatile("" ::"v"(raw));
      if (i + 1 < past) enter(i + 1, kept_next, next, raw);
    }
    kept = kept_next;
    wait_vmcnt<0>();
    __syncthreads();
  };
  if (from < to) {
    stage_k(from, 0);
    stage_v(from, 0);
    if (from + 1 < to) stage_k(from + 1, 1);
    wait_vmcnt<0>();
    __syncthreads();
    if (from < past) {
      clear(sa);
#pragma unroll
      for (int f = 0; f < 16; ++f) score(sa, key_frag(slot_k(0), f), f);
    }
    if (from + 2 < to) __syncthreads();  // K(from + 2) goes where K(from) was
    kept = kept_of(tile_of(from));
    if (from < past) enter(from, kept, sa, largest(sa));
    for (int i = from; i < to; i += 2) {
      step(i, std::integral_constant<int, 0>{}, sa, sb);
      if (i + 1 < to) step(i + 1, std::integral_constant<int, 1>{}, sb, sa);
    }
  }
  const float l = lane_sum32(l_run);
  const int parts = p.parts();
  if (c0 + col >= ncols) return;
  if (parts > 1) {
    float* const dst = part_sums(a, part, qh) + 4 * hi;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(dst + 32 * dt + 8 * g) = f32x4{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
    if (hi == 0) *reinterpret_cast<float2*>(part_stats(a, parts, part, qh)) = make_float2(m_run, l);
    return;
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  bf16_t* const dst = a.out + qh * PA_DH + 4 * hi;
  const int row = (int)(qh / a.H), first = (int)(qh % a.H) * PA_DH + 4 * hi;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float v[4] = {o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
      const u32x2 two = result4(v, inv);
      *reinterpret_cast<u32x2*>(dst + 32 * dt + 8 * g) = two;
      if (a.out_pack) *reinterpret_cast<u32x2*>(a.out_pack + pack_off(row, first + 32 * dt + 8 * g, a.H * PA_DH)) = two;
    }
}

// ---- 16 columns of one row and one wave, 32 keys a step: keys straight from memory into registers (lane's key lane & 15 of each 16, dims
// 32 j + 8 (lane >> 4) .. +7, the query's the same), values through two wave-private LDS slots. Steps [from, to) of the prefix's keys (where
// there are some) and the row's own after them. Lane (g, j) is left with dims 16 dt + 4 g .. + 3 of column j in o[dt].
struct WaveSums {
  f32x4 o[8];
  float m, l;
};
constexpr int PA_WAVE_LDS = 2 * PA_STEP * PA_DH * 2;

JLA_DEV void wave_columns(WaveSums& st, const PrefixAttn& a, size_t qh, int upto, const KeyRange& pre, const KeyRange& own, int from, int to, char* lds) {
  const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
  const float scale = 1.4426950408889634f / 11.313708498984761f;
  const int n_pre = pre.tiles(PA_STEP);
  u32x4 qf[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) qf[i] = *reinterpret_cast<const u32x4*>(a.q + qh * PA_DH + 32 * i + 8 * g);
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) st.o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  st.m = -INFINITY;
  st.l = 0.f;
  u32x4 kr[2][8];
  uint32_t kept[2];  // a bit for each of a step's keys that the range and the mask leave
  auto issue = [&](int i, u32x4 (&k)[8], uint32_t& bits, char* vd) {
    const bool is_own = i >= n_pre;
    const int t0 = is_own ? own.first(PA_STEP) + (i - n_pre) * PA_STEP : pre.first(PA_STEP) + i * PA_STEP;
    const int lo = is_own ? own.lo : pre.lo, hi = is_own ? own.hi : pre.hi, last = (is_own ? own.limit : pre.limit) - 1;
    const bf16_t* const kp = is_own ? own.k : pre.k;
    const bf16_t* const vp = is_own ? own.v : pre.v;
    const uint8_t* const mask = is_own ? nullptr : pre.mask;
    bits = ~0u;
    if (t0 < lo || t0 + PA_STEP > hi || mask) {
      const int key = t0 + (lane & 31);
      bits = (uint32_t)__ballot(key >= lo && key < hi && (!mask || mask[min(key, last)]));
    }
#pragma unroll
    for (int bi = 0; bi < 8; ++bi) {
      const int row = 4 * bi + g, ch = j ^ (((row & 3) << 2) | ((row >> 2) & 3));
      glds16_asm(vp + (size_t)t0 * PA_DH, 256 * min(row, last - t0) + 16 * ch, vd + 1024 * bi);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const bf16_t* const at = kp + (size_t)min(t0 + 16 * kk + j, last) * PA_DH + 8 * g;
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) k[4 * kk + i4] = *reinterpret_cast<const u32x4*>(at + 32 * i4);
    }
  };
  auto compute = [&](int i, const u32x4 (&k)[8], uint32_t bits, char* vt) {
    if (bits != ~0u) {  // values of keys that nobody attends may be anything: 0 x NaN would not be 0
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (!(bits >> (4 * q + g) & 1)) *reinterpret_cast<u32x4*>(vt + 1024 * q + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
      __builtin_amdgcn_wave_barrier();
    }
    f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      s[0] = mfma16x16x32(k[i4], qf[i4], s[0]);
      s[1] = mfma16x16x32(k[4 + i4], qf[i4], s[1]);
    }
    if (i >= n_pre) {  // a column's own keys end at its slot
      const int n = upto + 1 - (own.first(PA_STEP) + (i - n_pre) * PA_STEP);
      bits &= n >= PA_STEP ? ~0u : n > 0 ? (1u << n) - 1 : 0u;
    }
    bits >>= 4 * g;  // score e is key 16 (e >> 2) + 4 g + (e & 3) of the step
    float sc[8], most = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sc[e] = bits >> (16 * (e >> 2) + (e & 3)) & 1 ? s[e >> 2][e & 3] * scale : -INFINITY;
      most = fmaxf(most, sc[e]);
    }
    most = lane_max32(lane_max16(most));
    if (__ballot(most > st.m + 8.f)) {
      const float m_new = fmaxf(st.m, most);
      const float alpha = __builtin_amdgcn_exp2f(st.m - (m_new == -INFINITY ? 0.f : m_new));
      st.l *= alpha;
      st.m = m_new;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) st.o[dt] *= alpha;
    }
    const float m_use = st.m == -INFINITY ? 0.f : st.m;
    float e[8];
#pragma unroll
    for (int i8 = 0; i8 < 8; ++i8) {
      e[i8] = __builtin_amdgcn_exp2f(sc[i8] - m_use);
      st.l += e[i8];
    }
    const u32x4 pf = pack8(e);
    const int row = 4 * g + (j >> 2), pp = lane & 3;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      const int ch = 2 * dt + (pp >> 1);
      const u32x2 lo4 = ld_tr(vt, pa_off(row, ch) + 8 * (pp & 1)), hi4 = ld_tr(vt, pa_off(row + 16, ch) + 8 * (pp & 1));
      st.o[dt] = mfma16x16x32(u32x4{lo4[0], lo4[1], hi4[0], hi4[1]}, pf, st.o[dt]);
    }
  };
  char* const slot_a = lds;
  char* const slot_b = lds + PA_STEP * PA_DH * 2;
  if (from < to) issue(from, kr[0], kept[0], slot_a);
  for (int i = from; i < to; i += 2) {
    wait_vmcnt<0>();
    if (i + 1 < to) issue(i + 1, kr[1], kept[1], slot_b);
    compute(i, kr[0], kept[0], slot_a);
    if (i + 1 < to) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // slot a is read: it may be filled again
      wait_vmcnt<0>();
      if (i + 2 < to) issue(i + 2, kr[0], kept[0], slot_a);
      compute(i + 1, kr[1], kept[1], slot_b);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
  st.l = lane_sum32(lane_sum16(st.l));
}

// a wave's split of a row's own keys, beside the prefix's tiles
JLA_DEV void own_part(const PrefixAttn& a, const PrefixPlan& p, int split, int kvh, int b, int ct, char* lds) {
  const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
  const int ncols = a.S * a.rep, c0 = 16 * ct, c = min(c0 + j, ncols - 1);
  const size_t qh = ((size_t)b * a.S + c / a.rep) * a.H + kvh * a.rep + c % a.rep;
  const KeyRange own = own_keys(a, b, kvh, min(c0 + 15, ncols - 1) / a.rep);
  const int n = own.tiles(PA_STEP);
  WaveSums st;
  wave_columns(st, a, qh, own_slot(a) + c / a.rep, KeyRange{}, own, (int)((long long)n * split / p.own_ns), (int)((long long)n * (split + 1) / p.own_ns), lds);
  if (c0 + j >= ncols) return;
  float* const dst = part_sums(a, p.ns + split, qh) + 4 * g;
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(dst + 16 * dt) = st.o[dt];
  if (g == 0) *reinterpret_cast<float2*>(part_stats(a, p.parts(), p.ns + split, qh)) = make_float2(st.m, st.l);
}

// Short prefixes: one launch. A workgroup of eight waves takes 16 columns of a (row, kv head) over prefix and own keys, each wave an eighth of
// their steps; the waves' parts join in LDS.
constexpr int PS_WAVES = 8, PS_LDS = PS_WAVES * PA_WAVE_LDS;

__global__ void __launch_bounds__(64 * PS_WAVES, 2) prefix_short_kernel(PrefixAttn a, PrefixPlan p) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, j = lane & 15;
  int id = blockIdx.x;
  const int kvh = id % a.Hkv;
  id /= a.Hkv;
  const int ct = id % p.own_ct, b = id / p.own_ct;
  const int ncols = a.S * a.rep, c0 = 16 * ct, c = min(c0 + j, ncols - 1);
  const size_t row0 = (size_t)b * a.S;
  const KeyRange pre = prefix_keys(a, b / a.n, kvh), own = own_keys(a, b, kvh, min(c0 + 15, ncols - 1) / a.rep);
  const int n = pre.tiles(PA_STEP) + own.tiles(PA_STEP);
  WaveSums st;
  wave_columns(st, a, (row0 + c / a.rep) * a.H + kvh * a.rep + c % a.rep, own_slot(a) + c / a.rep, pre, own, n * w / PS_WAVES, n * (w + 1) / PS_WAVES,
               lds + w * PA_WAVE_LDS);
  // [32 chunks of 4 dims][16 columns and one for the banks] sums, then the statistics, in each wave's share
  auto sums = [&](int wave) { return reinterpret_cast<f32x4*>(lds + wave * PA_WAVE_LDS); };
  auto stats = [&](int wave) { return reinterpret_cast<float2*>(lds + wave * PA_WAVE_LDS + 32 * 17 * 16); };
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) sums(w)[(4 * dt + g) * 17 + j] = st.o[dt];
  if (g == 0) stats(w)[j] = make_float2(st.m, st.l);
  __syncthreads();
  const int oc = tid >> 5, q = tid & 31;  // its column and chunk
  if (c0 + oc >= ncols) return;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < PS_WAVES; ++i) m = fmaxf(m, stats(i)[oc].x);
  const float m_use = m == -INFINITY ? 0.f : m;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < PS_WAVES; ++i) {
    const float2 s = stats(i)[oc];
    const float f = __builtin_amdgcn_exp2f(s.x - m_use);
    l += f * s.y;
    o += f * sums(i)[q * 17 + oc];
  }
  const float v[4] = {o[0], o[1], o[2], o[3]};
  const u32x2 two = result4(v, l != 0.f ? 1.f / l : 0.f);
  const size_t row = row0 + (c0 + oc) / a.rep;
  const int d = (kvh * a.rep + (c0 + oc) % a.rep) * PA_DH + 4 * q;
  *reinterpret_cast<u32x2*>(a.out + row * a.H * PA_DH + d) = two;
  if (a.out_pack) *reinterpret_cast<u32x2*>(a.out_pack + pack_off((int)row, d, a.H * PA_DH)) = two;
}

// One launch: workgroups [0, tiles) take 128 columns each, the others a wave per (row, kv head, 16 columns, split) of own keys.
__global__ void __launch_bounds__(256, 2) prefix_attn_kernel(PrefixAttn a, PrefixPlan p, int tiles, int own_waves) {
  __shared__ __attribute__((aligned(16))) char lds[4 * PA_TILE];
  const int rep = a.rep, n = a.n;
  if ((int)blockIdx.x < tiles) {
    // Kv heads first, then columns: where kv heads are a multiple of the 8 XCDs, all tiles that read the same keys run on one of them,
    // behind one L2, and at the same time (64 rows behind 65536 keys, two tiles of columns: 91 us, 101 with the keys' parts first).
    int id = blockIdx.x;
    const int kvh = id % a.Hkv;
    id /= a.Hkv;
    const int ct = id % p.ct;
    id /= p.ct;
    const int part = id % p.ns, u = id / p.ns;
    const int ncols = (p.by_row ? 1 : n) * a.S * rep;
    KeyRange own = own_keys(a, u, kvh, (min(ncols, (ct + 1) * PA_COLS) - 1) / rep);  // (by a group's number: row u exists too)
    if (!p.by_row) own.hi = own.lo;
    column_tile(a, p, part, kvh, (size_t)u * (p.by_row ? 1 : n) * a.S, ncols, ct, prefix_keys(a, p.by_row ? u / n : u, kvh), own, lds);
    return;
  }
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = ((int)blockIdx.x - tiles) * 4 + w;
  if (id >= own_waves) return;
  const int ct = id % p.own_ct;
  id /= p.own_ct;
  const int split = id % p.own_ns;
  id /= p.own_ns;
  own_part(a, p, split, id % a.Hkv, id / a.Hkv, ct, lds + w * PA_WAVE_LDS);
}

// The parts of a (token, head) join in their order: 8 groups of 32 lanes (4 dims each) take every eighth part, so that their loads are
// under way together, and add up in LDS: 34 MB of 33 parts of 64 rows of 32 heads 10 us, 3 MB 4 us.
__global__ void __launch_bounds__(256) prefix_join_kernel(PrefixAttn a, int parts) {
  __shared__ f32x4 so[8][32];
  __shared__ float sl[8];
  const size_t n = (size_t)a.B * a.S * a.H, qh = blockIdx.x;
  const int g = threadIdx.x >> 5, d = 4 * (threadIdx.x & 31);
  const float* ml = part_stats(a, parts, 0, qh);
  float m = -INFINITY;
  for (int i = threadIdx.x & 31; i < parts; i += 32) m = fmaxf(m, ml[2 * n * i]);
#pragma unroll
  for (int j = 1; j < 32; j <<= 1) m = fmaxf(m, __shfl_xor(m, j, 64));
  const float m_use = m == -INFINITY ? 0.f : m;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int i = g; i < parts; i += 8) {
    const float2 s = *reinterpret_cast<const float2*>(ml + 2 * n * i);
    const float f = __builtin_amdgcn_exp2f(s.x - m_use);
    l += f * s.y;
    o += f * *reinterpret_cast<const f32x4*>(a.part + (n * i + qh) * PA_DH + d);
  }
  so[g][d >> 2] = o;
  if (d == 0) sl[g] = l;
  __syncthreads();
  if (g) return;
  const int groups = min(parts, 8);
  for (int i = 1; i < groups; ++i) {
    o += so[i][d >> 2];
    l += sl[i];
  }
  const float v[4] = {o[0], o[1], o[2], o[3]};
  const u32x2 two = result4(v, l != 0.f ? 1.f / l : 0.f);
  *reinterpret_cast<u32x2*>(a.out + qh * PA_DH + d) = two;
  if (a.out_pack) *reinterpret_cast<u32x2*>(a.out_pack + pack_off((int)(qh / a.H), (int)(qh % a.H) * PA_DH + d, a.H * PA_DH)) = two;
}

static int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Which queries share a workgroup, and how the keys are split.
//
// A row's own columns go over prefix and own keys together (by_row), or a group's over the prefix with the own keys beside; each with the
// fewest splits of the least time by this model, in us: a tile takes 1.05 where a compute unit has one workgroup and 1.65 where it has two,
// in rounds of 512; a wave's step of own keys 1.2 beside those, and 0.6 with 2048 under way; each part's sums are written and read at about 4.5 TB/s, and their
// join costs a launch. Measured, by splits: 32 rows behind 2048 tokens 16.0 with 8 and 12 (4: 18.3, 32: 18.7), 200 behind 16384 72 with 9
// (4: 79, 12: 88), 1000 queries of one row behind 8000 152 with 1 (2: 161, 3: 185). Shared | by row, 16 rows behind 4096 tokens: 16 columns
// each 21.7 | 39, 64 36.7 | 48, 144 62.8 | 71.6, 192 80 | 70; 64 rows of 100 columns behind 1000 79 | 40.5; a row alone is by
// row (behind 32768 tokens with 2000 of its own 36 | 29, 8 of them behind 8192 45.7 | 44.8).
static PrefixPlan plan_of(int B, int S, int H, int Hkv, int G, int P, int T, bool by_row, double& best) {
  PrefixPlan p{};
  const int rep = H / Hkv, n = B / G;
  p.by_row = by_row;
  const long long cols = (long long)(by_row ? 1 : n) * S * rep;
  const int keys = ceil_div(P, PA_KT) + (by_row ? ceil_div(T, PA_KT) : 0);
  p.ct = (int)((cols + PA_COLS - 1) / PA_COLS);
  const long long tiles = (long long)(by_row ? B : G) * Hkv * p.ct;
  const double part = 2. * 4 * (PA_DH + 2) * B * S * H / 4.5e6;
  auto tiles_time = [&](int ns) {
    const long long groups = tiles * ns, rest = groups % 512;
    return ceil_div(keys, ns) * ((double)(groups / 512) * 1.65 + (rest == 0 ? 0. : rest <= 256 ? 1.05 : 1.65));
  };
  best = 1e30;
  for (int ns = 1; ns <= keys && (ns == 1 || tiles * ns <= 1024); ++ns) {
    const double t = tiles_time(ns) + (by_row && ns == 1 ? 0. : part * ns + 3.5);
    if (t < best) best = t, p.ns = ns;
  }
  if (!by_row) {  // own keys as long as the prefix's tiles run, or 3 us
    p.own_ct = ceil_div(S * rep, 16);
    const double steps = ceil_div(T, PA_STEP), beside = tiles_time(p.ns) > 3. ? tiles_time(p.ns) : 3.;
    const long long waves = (long long)B * Hkv * p.own_ct, most = waves >= 2048 ? 1 : 2048 / waves;
    const long long want = (long long)(1.2 * steps / beside) + 1;
    p.own_ns = (int)(want < most ? want : most);
    best += part * p.own_ns + 0.6 * steps * waves / 2048;
  }
  return p;
}

PrefixPlan prefix_attn_plan(int B, int S, int H, int Hkv, int G, int P, int T) {
  double best, by_row;
  PrefixPlan p = plan_of(B, S, H, Hkv, G, P, T, false, best);
  const PrefixPlan rows = plan_of(B, S, H, Hkv, G, P, T, true, by_row);
  if (B == G || by_row < best) p = rows, best = by_row;
  // Short ones in one launch, 16 columns a workgroup: a step of its eight waves takes about 2 us (128 KiB through one compute unit), less in
  // several rounds; the two launches take some 0.6 us more than the sum above. One | two launches, us: 2 rows behind 130 tokens 5.5 | 9.3, 32
  // behind 250 7.2 | 10.5, 32 behind 700 10.5 | 13.4, 8 of 8 queries behind 300 7.9 | 11.0, 8 behind 700 10.3 | 9.6, 4 behind 1000 13.3 | 9.5, 128 behind
  // 130 18.1 | 16.0, 8 of 64 queries behind 200 24.6 | 12.8.
  const int rows_ct = ceil_div(S * (H / Hkv), 16), steps = ceil_div(ceil_div(P, PA_STEP) + ceil_div(T, PA_STEP), PS_WAVES);
  const long long rounds = ((long long)B * Hkv * rows_ct + 255) / 256;
  if ((rounds == 1 ? 2. * steps : 1.5 * rounds * (steps + 1)) < best + 0.6) p.brief = 1, p.own_ct = rows_ct;
  return p;
}

long long prefix_attn_workspace(const PrefixPlan& p, int B, int S, int H) {
  return !p.brief && p.parts() > 1 ? (long long)p.parts() * B * S * H * (PA_DH + 2) : 0;
}

int prefix_attn(const PrefixAttn& a, const PrefixPlan& p, hipStream_t s) {
  if (a.B <= 0 || a.S <= 0) return 0;
  if (a.H % a.Hkv || a.G <= 0 || a.B % a.G || a.P < 1 || a.T < 1) return -1;
  if (p.brief) {
    static std::atomic<unsigned long long> has_room{0};  // a bit for each of the first devices: the limit is a device's
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return (int)e;
    if (device >= 64 || !(has_room.load() >> device & 1)) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(prefix_short_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, PS_LDS);
      if (e != hipSuccess) return (int)e;
      if (device < 64) has_room |= 1ull << device;
    }
    const long long items = (long long)a.B * a.Hkv * p.own_ct;
    if (items > 0x7fffffff) return -3;
    prefix_short_kernel<<<(int)items, 64 * PS_WAVES, PS_LDS, s>>>(a, p);
    return (int)hipGetLastError();
  }
  const int parts = p.parts();
  if (parts > 1 && !a.part) return -2;
  const long long tiles = (long long)(p.by_row ? a.B : a.G) * a.Hkv * p.ct * p.ns;
  const long long own_waves = p.by_row ? 0 : (long long)a.B * a.Hkv * p.own_ct * p.own_ns;
  const long long grid = tiles + (own_waves + 3) / 4, join = (long long)a.B * a.S * a.H;
  if (grid > 0x7fffffff || own_waves > 0x7ffffff0 || join > 0x7fffffff) return -3;
  prefix_attn_kernel<<<(int)grid, 256, 0, s>>>(a, p, (int)tiles, (int)own_waves);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (parts > 1) {
    prefix_join_kernel<<<(int)join, 256, 0, s>>>(a, parts);
    e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}

}  // namespace jla
