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
#include "../kernels/common.h"
#include "serving.h"

namespace jla {

constexpr int PA_DH = 128;
constexpr int PA_KT = 64;                         // keys per tile of a workgroup's 128 columns
constexpr int PA_TILE = PA_KT * PA_DH * 2;        // 16 KiB
constexpr int PA_STEP = 32;                       // keys per step of a wave's 16 columns
constexpr int PA_COLS = 128;

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
  r.hi = min(a.slot[0] + s_last + 1, a.T);
  r.limit = a.T;
  r.mask = nullptr;
  return r;
}

// One part of a query head: the sums (4 of its dims from d on per call), or where there is one part the result
JLA_DEV void put_sums(const PrefixAttn& a, int part, size_t qh, int d, const float* o) {
  *reinterpret_cast<f32x4*>(a.part + ((size_t)part * a.B * a.S * a.H + qh) * PA_DH + d) = f32x4{o[0], o[1], o[2], o[3]};
}
JLA_DEV void put_stats(const PrefixAttn& a, int parts, int part, size_t qh, float m, float l) {
  const size_t n = (size_t)a.B * a.S * a.H;
  *reinterpret_cast<float2*>(a.part + n * PA_DH * parts + (part * n + qh) * 2) = make_float2(m, l);
}
JLA_DEV void put_result(const PrefixAttn& a, size_t qh, int d, const float* o, float inv) {
  const u32x2 v = {pack2bf(o[0] * inv, o[1] * inv), pack2bf(o[2] * inv, o[3] * inv)};
  *reinterpret_cast<u32x2*>(a.out + qh * PA_DH + d) = v;
  if (a.out_pack) {
    const int K = a.H * PA_DH;
    *reinterpret_cast<u32x2*>(a.out_pack + pack_off((int)(qh / a.H), (int)(qh % a.H) * PA_DH + d, K)) = v;
  }
}

// ---- 128 columns of a workgroup of four waves, 32 a wave (a lane's column is lane & 31). Tiles of 64 keys go to LDS by LDS-DMA, two
// slots each for keys and values; S^T = K Q^T leaves a column's scores in its two lanes, which are the operand of O^T += V^T P^T as
// they are (V^T by transposing reads).
JLA_DEV void column_tile(const PrefixAttn& a, const PrefixPlan& p, int part, int kvh, size_t tok0, int ncols, int ct, const KeyRange& pre,
                         const KeyRange& own, char* lds) {
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, rep = a.H / a.Hkv;
  const int c0 = ct * PA_COLS + 32 * w, c = min(c0 + (lane & 31), ncols - 1);
  const bool active = c0 < ncols;  // (the wave's; the others help to stage)
  const size_t qh = (tok0 + c / rep) * a.H + kvh * rep + c % rep;
  const float scale = 1.4426950408889634f / 11.313708498984761f;
  // its slot; that of the wave's first column
  const int slot = a.slot[0], at = slot + c / rep, at_first = slot + min(c0, ncols - 1) / rep;

  u32x4 qf[8];
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) qf[ks] = *reinterpret_cast<const u32x4*>(a.q + qh * PA_DH + 16 * ks + 8 * hi);
  f32x16 o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  const int n_pre = pre.tiles(PA_KT), n_all = n_pre + own.tiles(PA_KT);
  const int from = (int)((long long)n_all * part / p.ns), to = (int)((long long)n_all * (part + 1) / p.ns);
  auto stage = [&](int i) {
    const bool is_own = i >= n_pre;
    const KeyRange& r = is_own ? own : pre;
    const int t0 = r.first(PA_KT) + (is_own ? i - n_pre : i) * PA_KT;
    char* const kd = lds + (i & 1) * PA_TILE;
    char* const vd = lds + (2 + (i & 1)) * PA_TILE;
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // 1-KiB blocks of 4 rows; lane L fills row L / 16, place L % 16 of its block
      const int bi = w + 4 * j, row = 4 * bi + (lane >> 4);
      const int ch = (lane & 15) ^ (((row & 3) << 2) | ((row >> 2) & 3));
      const int off = 256 * min(row, r.limit - 1 - t0) + 16 * ch;
      glds16_asm(r.k + (size_t)t0 * PA_DH, off, kd + 1024 * bi);
      glds16_asm(r.v + (size_t)t0 * PA_DH, off, vd + 1024 * bi);
    }
  };
  const int col = lane & 31, gq = (lane & 15) >> 2, gp = lane & 3, G = lane >> 4;
  if (from < to) stage(from);
  wait_vmcnt<0>();
  __syncthreads();
  for (int i = from; i < to; ++i) {
    if (i + 1 < to) stage(i + 1);
    const bool is_own = i >= n_pre;
    const KeyRange& r = is_own ? own : pre;
    const int t0 = r.first(PA_KT) + (is_own ? i - n_pre : i) * PA_KT;
    const char* const kt = lds + (i & 1) * PA_TILE;
    char* const vt = lds + (2 + (i & 1)) * PA_TILE;
    const bool edge = t0 < r.lo || t0 + PA_KT > r.hi || r.mask;  // (the workgroup's)
    if (edge) {  // values of keys that nobody attends may be anything: 0 x NaN would not be 0
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = (tid >> 4) + 16 * j, key = t0 + row;
        if (key < r.lo || key >= r.hi || (r.mask && !r.mask[key]))
          *reinterpret_cast<u32x4*>(vt + 256 * row + 16 * (tid & 15)) = u32x4{0u, 0u, 0u, 0u};
      }
      __syncthreads();
    }
    if (active) {
      f32x16 s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          s[kb] = mfma32(*reinterpret_cast<const u32x4*>(kt + pa_off(32 * kb + col, 2 * ks + hi)), qf[ks], s[kb]);
      }
      // element e of block kb is key t0 + 32 kb + (e & 3) + 8 (e >> 2) + 4 hi
      if (edge || (is_own && t0 + PA_KT - 1 > at_first)) {
        const int upto = is_own ? min(at, r.hi - 1) : r.hi - 1;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = t0 + 32 * kb + (e & 3) + 8 * (e >> 2) + 4 * hi;
            bool ok = key >= r.lo && key <= upto;
            if (r.mask) ok = ok && r.mask[min(key, r.limit - 1)];
            s[kb][e] = ok ? s[kb][e] : -INFINITY;
          }
      }
      float most = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) most = fmaxf(most, s[kb][e]);
      most = lane_max32(most) * scale;
      // the maximum moves, and the sums with it, only where it grew by more than 8: 2^(x - m) stays below 256
      if (__ballot(most > m_run + 8.f)) {
        const float m_new = fmaxf(m_run, most);
        const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
        l_run *= alpha;
        m_run = m_new;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
      }
      const float m_use = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] = __builtin_amdgcn_exp2f(fmaf(s[ks >> 1][8 * (ks & 1) + j], scale, -m_use));
          l_run += e[j];
        }
        const u32x4 pf = pack8(e);  // (bf16 weights for the matrix cores: 2^-9 of each, their sum is of the unrounded ones)
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
          const int row = 16 * ks + 4 * (G >> 1) + gq, ch = 4 * dt + 2 * (G & 1) + (gp >> 1);
          const u32x2 lo4 = ld_tr(vt, pa_off(row, ch) + 8 * (gp & 1)), hi4 = ld_tr(vt, pa_off(row + 8, ch) + 8 * (gp & 1));
          o[dt] = mfma32(u32x4{lo4[0], lo4[1], hi4[0], hi4[1]}, pf, o[dt]);
        }
      }
    }
    wait_vmcnt<0>();
    __syncthreads();
  }
  l_run = lane_sum32(l_run);
  if (c0 + col >= ncols) return;
  const int parts = p.parts();
  const float inv = l_run != 0.f ? 1.f / l_run : 0.f;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float v[4] = {o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
      if (parts > 1) put_sums(a, part, qh, 32 * dt + 8 * g + 4 * hi, v);
      else put_result(a, qh, 32 * dt + 8 * g + 4 * hi, v, inv);
    }
  if (parts > 1 && hi == 0) put_stats(a, parts, part, qh, m_run, l_run);
}

// ---- 16 columns of one wave over its row's own keys, 32 a step: keys straight from memory into registers (lane's key lane & 15 of each
// 16, dims 32 j + 8 (lane >> 4) .. +7, the query's the same), values through two wave-private LDS slots.
JLA_DEV void own_step_columns(const PrefixAttn& a, const PrefixPlan& p, int split, int kvh, int b, int ct, char* lds) {
  const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
  const int rep = a.H / a.Hkv, ncols = a.S * rep;
  const int c0 = 16 * ct, c = min(c0 + j, ncols - 1);
  const size_t qh = ((size_t)b * a.S + c / rep) * a.H + kvh * rep + c % rep;
  const float scale = 1.4426950408889634f / 11.313708498984761f;
  const KeyRange r = own_keys(a, b, kvh, min(c0 + 15, ncols - 1) / rep);
  const int upto = min(a.slot[0] + c / rep, r.hi - 1);
  const int n = r.tiles(PA_STEP);
  const int from = (int)((long long)n * split / p.own_ns), to = (int)((long long)n * (split + 1) / p.own_ns);
  u32x4 qf[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) qf[i] = *reinterpret_cast<const u32x4*>(a.q + qh * PA_DH + 32 * i + 8 * g);
  f32x4 o[8];
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;
  u32x4 kr[2][8];
  auto issue = [&](int i, u32x4 (&k)[8], char* vd) {
    const int t0 = r.first(PA_STEP) + i * PA_STEP;
#pragma unroll
    for (int bi = 0; bi < 8; ++bi) {
      const int row = 4 * bi + g, ch = j ^ (((row & 3) << 2) | ((row >> 2) & 3));
      glds16_asm(r.v + (size_t)min(t0 + row, r.limit - 1) * PA_DH + 8 * ch, vd + 1024 * bi);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4)
        k[4 * kk + i4] = *reinterpret_cast<const u32x4*>(r.k + (size_t)min(t0 + 16 * kk + j, r.limit - 1) * PA_DH + 32 * i4 + 8 * g);
  };
  auto compute = [&](int i, const u32x4 (&k)[8], char* vt) {
    const int t0 = r.first(PA_STEP) + i * PA_STEP;
    const bool edge = t0 < r.lo || t0 + PA_STEP > r.hi;
    if (edge) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int row = 4 * q + g, key = t0 + row;
        if (key < r.lo || key >= r.hi) *reinterpret_cast<u32x4*>(vt + 256 * row + 16 * j) = u32x4{0u, 0u, 0u, 0u};
      }
      __builtin_amdgcn_wave_barrier();
    }
    f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      s[0] = mfma16x16x32(k[i4], qf[i4], s[0]);
      s[1] = mfma16x16x32(k[4 + i4], qf[i4], s[1]);
    }
    float sc[8];  // keys t0 + 4 g + e, and + 16
    float most = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int key = t0 + 16 * (e >> 2) + 4 * g + (e & 3);
      sc[e] = key >= r.lo && key <= upto ? s[e >> 2][e & 3] * scale : -INFINITY;
      most = fmaxf(most, sc[e]);
    }
    most = lane_max32(lane_max16(most));
    if (__ballot(most > m_run + 8.f)) {
      const float m_new = fmaxf(m_run, most);
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
      l_run *= alpha;
      m_run = m_new;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) o[dt] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    float e[8];
#pragma unroll
    for (int i8 = 0; i8 < 8; ++i8) {
      e[i8] = __builtin_amdgcn_exp2f(sc[i8] - m_use);
      l_run += e[i8];
    }
    const u32x4 pf = pack8(e);
    const int row = 4 * g + (j >> 2), pp = lane & 3;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      const int ch = 2 * dt + (pp >> 1);
      const u32x2 lo4 = ld_tr(vt, pa_off(row, ch) + 8 * (pp & 1)), hi4 = ld_tr(vt, pa_off(row + 16, ch) + 8 * (pp & 1));
      o[dt] = mfma16x16x32(u32x4{lo4[0], lo4[1], hi4[0], hi4[1]}, pf, o[dt]);
    }
  };
  char* const slot_a = lds;
  char* const slot_b = lds + PA_STEP * PA_DH * 2;
  if (from < to) issue(from, kr[0], slot_a);
  for (int i = from; i < to; i += 2) {
    wait_vmcnt<0>();
    if (i + 1 < to) issue(i + 1, kr[1], slot_b);
    compute(i, kr[0], slot_a);
    if (i + 1 < to) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // slot a is read: it may be filled again
      wait_vmcnt<0>();
      if (i + 2 < to) issue(i + 2, kr[0], slot_a);
      compute(i + 1, kr[1], slot_b);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
  l_run = lane_sum32(lane_sum16(l_run));
  if (c0 + j >= ncols) return;
  const int parts = p.parts(), part = p.ns + split;
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) {
    const float v[4] = {o[dt][0], o[dt][1], o[dt][2], o[dt][3]};
    put_sums(a, part, qh, 16 * dt + 4 * g, v);
  }
  if (g == 0) put_stats(a, parts, part, qh, m_run, l_run);
}

// One launch: workgroups [0, tiles) take 128 columns each, the others a wave per (row, kv head, 16 columns, split) of own keys.
__global__ void __launch_bounds__(256, 2) prefix_attn_kernel(PrefixAttn a, PrefixPlan p, int tiles, int own_waves) {
  __shared__ __attribute__((aligned(16))) char lds[4 * PA_TILE];
  const int rep = a.H / a.Hkv, n = a.B / a.G;
  if ((int)blockIdx.x < tiles) {
    int id = blockIdx.x;
    const int ct = id % p.ct;
    id /= p.ct;
    const int part = id % p.ns;
    id /= p.ns;
    const int kvh = id % a.Hkv, u = id / a.Hkv;
    if (p.by_row) {
      const int ncols = a.S * rep;
      column_tile(a, p, part, kvh, (size_t)u * a.S, ncols, ct, prefix_keys(a, u / n, kvh),
                  own_keys(a, u, kvh, (min(ncols, (ct + 1) * PA_COLS) - 1) / rep), lds);
    } else {
      KeyRange none{};
      column_tile(a, p, part, kvh, (size_t)u * n * a.S, n * a.S * rep, ct, prefix_keys(a, u, kvh), none, lds);
    }
    return;
  }
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = ((int)blockIdx.x - tiles) * 4 + w;
  if (id >= own_waves) return;
  const int ct = id % p.own_ct;
  id /= p.own_ct;
  const int split = id % p.own_ns;
  id /= p.own_ns;
  own_step_columns(a, p, split, id % a.Hkv, id / a.Hkv, ct, lds + w * PA_TILE);
}

// 32 lanes per (token, head), four of its dims each: the parts join in their order
__global__ void __launch_bounds__(256) prefix_join_kernel(PrefixAttn a, int parts) {
  const size_t n = (size_t)a.B * a.S * a.H, qh = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (qh >= n) return;
  const int d = 4 * (threadIdx.x & 31);
  const float* ml = a.part + n * PA_DH * parts + qh * 2;
  float m = -INFINITY;
  for (int i = 0; i < parts; ++i) m = fmaxf(m, ml[2 * n * i]);
  const float m_use = m == -INFINITY ? 0.f : m;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (int i = 0; i < parts; ++i) {
    const float2 s = *reinterpret_cast<const float2*>(ml + 2 * n * i);
    const float f = __builtin_amdgcn_exp2f(s.x - m_use);
    l += f * s.y;
    o += f * *reinterpret_cast<const f32x4*>(a.part + (n * i + qh) * PA_DH + d);
  }
  const float v[4] = {o[0], o[1], o[2], o[3]};
  put_result(a, qh, d, v, l != 0.f ? 1.f / l : 0.f);
}

static int ceil_div(int a, int b) { return (a + b - 1) / b; }

PrefixPlan prefix_attn_plan(int B, int S, int H, int Hkv, int G, int P, int T) {
  PrefixPlan p{};
  const int rep = H / Hkv, n = B / G;
  const int pre = ceil_div(P, PA_KT), own = ceil_div(T, PA_KT);
  p.by_row = S * rep >= 96;
  const int cols = p.by_row ? S * rep : n * S * rep;
  p.ct = ceil_div(cols, PA_COLS);
  const long long tiles = (long long)(p.by_row ? B : G) * Hkv * p.ct;
  const int keys = p.by_row ? pre + own : pre;
  const long long want = tiles >= 384 ? 1 : (512 + tiles - 1) / tiles;
  p.ns = (int)(want < 1 ? 1 : want > (keys + 1) / 2 ? (keys + 1) / 2 : want);
  if (p.ns < 1) p.ns = 1;
  if (!p.by_row) {
    p.own_ct = ceil_div(S * rep, 16);
    const long long waves = (long long)B * Hkv * p.own_ct;
    const int steps = ceil_div(T, PA_STEP);
    const long long w = waves >= 1024 ? 1 : (1024 + waves - 1) / waves;
    p.own_ns = (int)(w > (steps + 3) / 4 ? (steps + 3) / 4 : w);
    if (p.own_ns < 1) p.own_ns = 1;
  }
  return p;
}

long long prefix_attn_workspace(const PrefixPlan& p, int B, int S, int H) {
  return p.parts() > 1 ? (long long)p.parts() * B * S * H * (PA_DH + 2) : 0;
}

int prefix_attn(const PrefixAttn& a, const PrefixPlan& p, hipStream_t s) {
  if (a.B <= 0 || a.S <= 0) return 0;
  if (a.H % a.Hkv || a.G <= 0 || a.B % a.G || a.P < 1 || a.T < 1) return -1;
  const int parts = p.parts();
  if (parts > 1 && !a.part) return -2;
  const long long tiles = (long long)(p.by_row ? a.B : a.G) * a.Hkv * p.ct * p.ns;
  const long long own_waves = p.by_row ? 0 : (long long)a.B * a.Hkv * p.own_ct * p.own_ns;
  const long long grid = tiles + (own_waves + 3) / 4, join = ((long long)a.B * a.S * a.H + 7) / 8;
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
