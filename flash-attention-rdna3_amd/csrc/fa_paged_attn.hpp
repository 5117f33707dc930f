// fa_paged_attn.hpp - attention over a paged cache whose codes have a scale for
// each block and head, over all blocks of a sequence or over listed ones.
//
//   S_rj = softmax_scale * ks[page(j)] * (q_r . k_j),   O_r = sum_j p_rj vs[page(j)] v_j / sum_j p_rj,
//   p_rj = exp(S_rj - m_r)
//
// One pass over the keys with a running maximum and sum, fp32 throughout.
//
//  * Work.  The keys of all sequences are one line of 32-key chunks, cut into
//    equal shares, one for each workgroup of a (KV head, row block): no
//    workgroup has more than another, whatever the lengths.  A share holds the
//    end of one sequence, whole ones, and the start of another; sequences that
//    several shares hold are merged from unnormalised partials by the last
//    workgroup that arrives (or by a second launch).
//  * Registers.  A wave streams its chunks through NBUF slots: K in the
//    layout of the matrix instruction's A operand, V as raw 16-byte pieces
//    that pass through an LDS tile of the wave and come back transposed.
//    Page ids and scales are scalar loads, so that they do not wait behind the
//    stream.  A slot is refilled right after its use.
//  * Types.  8-bit codes are fp16 numbers exactly, so over 8-bit caches the
//    products run in fp16 whatever the query's type: a bfloat16 query row is
//    scaled by a power of two to a largest value of 2^14 first (its 8 bits fit;
//    what is 2^-28 of the row's largest value loses bits).  ks joins the logit
//    scale.  p is rounded to fp16 with vs / vref on it, vref the largest power
//    of two seen over the scales: at most 2^8, and relative to what dominates.
//  * The maximum moves only when a logit passes it by more than 8 (in powers
//    of two): p <= 2^8 is exact enough in fp16, and most chunks then skip the
//    rescaling.
#pragma once

#include "fa_internal.hpp"
#include "fa_tiles.hpp"

namespace fa {

typedef float f32x4a __attribute__((ext_vector_type(4)));
typedef short s4a __attribute__((ext_vector_type(4)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));

struct PagedAttnArgs {
  const void* q;
  int64_t q_stride[3];  // batch, head, row
  void* out;
  int64_t out_stride[3];
  const void* k;
  const void* v;
  int64_t k_stride[3];  // block, position, head
  int64_t v_stride[3];
  const int32_t* table;
  int64_t table_stride[2];
  const int32_t* lens;
  int64_t lens_stride;
  const float* ks;
  const float* vs;
  int64_t ks_stride[2];  // block, head
  int64_t vs_stride[2];
  const int32_t* index;  // NULL: all blocks
  int64_t index_stride[3];
  int32_t n_index, num_blocks, max_blocks, shift;
  int32_t batch, heads_q, heads_kv, seqlen_q, bf16;
  float scale_log2;
  int32_t causal;
  int32_t shares;        // workgroups of a (head group, row block)
  int32_t head_shift;    // log2 of the KV heads of a workgroup
  float* ws_o;           // [2 * shares][heads_kv][row blocks][rows of a block][D]
  float* ws_ml;          // the same without D, pairs (m, l)
  uint32_t* tickets;
};

template <typename Tag, int KV, int D, int R, bool SMALL>
struct AttnCfg {
  static constexpr bool KV8 = KV != FA_KV_SAME;
  static constexpr int NW = (R >= 4 || D == 512 || !KV8) ? 4 : 8;  // waves
  static constexpr int NT = 64 * NW;
  static constexpr int NSTEP = D / 32;                        // 32-dim steps of Q K^T
  static constexpr int NDB = D / 16;                          // 16-dim blocks of O
  static constexpr bool PAIR = KV8 && NSTEP > 1;              // one 16-byte K load for two steps
  static constexpr int KN = PAIR ? NSTEP / 2 : NSTEP;         // K loads per 16 keys
  static constexpr int KREGS = KV8 && !PAIR ? 2 : 4;          // registers of one
  static constexpr int EPP = KV8 ? 16 : 8;                    // elements of a 16-byte V piece
  static constexpr int PPR = D / EPP;                         // pieces of a row
  static constexpr int VN = 32 * PPR / 64;                    // V loads per chunk
  static constexpr int SLOT = 2 * KN * KREGS + 4 * VN;
  // V of a 16-bit chunk at D = 512 loads at its use: no room for it beside K.
  static constexpr bool VLATE = !KV8 && D == 512;
  static constexpr int BUDGET = KV8 ? 64 : 128;
  static constexpr int NBUF = SLOT >= BUDGET ? 1 : BUDGET / SLOT > 4 ? 4 : BUDGET / SLOT;
  static constexpr int TILE_BYTES = 32 * D * 2;
  static constexpr int STATE = NDB * 4 + 2;                   // floats of a wave's row block per lane
  static constexpr int MERGE_BYTES = NW / 2 * R * STATE * 256;
  static constexpr int LOOP_BYTES = NW * TILE_BYTES;
  static constexpr int LDS_BYTES = (LOOP_BYTES > MERGE_BYTES ? LOOP_BYTES : MERGE_BYTES) + 16;
};

template <typename Tag> __device__ inline f32x4a mma16x16(s16x8 a, s16x8 b, f32x4a c);
template <> __device__ inline f32x4a mma16x16<f16_t>(s16x8 a, s16x8 b, f32x4a c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
}
template <> __device__ inline f32x4a mma16x16<bf16_t>(s16x8 a, s16x8 b, f32x4a c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}

// Eight int8 codes as fp16, exactly: 1024 + (x + 128) is the fp16 number with
// bits 0x6400 + (x + 128); subtract 1152.
__device__ inline s16x8 int8x8_to_f16(u32x2 r) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t u = r[i] ^ 0x80808080u;
    const h16x2 c = {(_Float16)1152.f, (_Float16)1152.f};
    o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - c);
    o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - c);
  }
  return __builtin_bit_cast(s16x8, u32x4{o[0], o[1], o[2], o[3]});
}

template <int KV> __device__ inline s16x8 codes_to_f16(u32x2 r) {
  if constexpr (KV == FA_KV_INT8) return int8x8_to_f16(r);
  else return fp8x8_to_op<f16_t>(r);
}

constexpr float kFloor = -3.0e38f;  // the running maximum before any key

// How the chunks of a (head group, row block) are shared out: `total` chunks
// over `count` workgroups, the first `extra` of them with one more.
struct Shares {
  int total, count, per, extra;
  __device__ int begin(int j) const { return j * per + min(j, extra); }
  __device__ int owner(int c) const {
    const int big = extra * (per + 1);
    return c < big ? c / (per + 1) : extra + (c - big) / per;
  }
};

struct PagedWork {
  const PagedAttnArgs& a;
  int rb_rows, rb;  // rows of a row block, and the row block
  __device__ int length(int b) const {
    const int64_t cap = min((int64_t)a.max_blocks << a.shift, (int64_t)INT_MAX);
    return (int)min((int64_t)max(a.lens[b * a.lens_stride], 0), cap);
  }
  // Chunks of sequence b: at least one, whose workgroup writes the rows of an
  // empty sequence.  Keys behind the last one that any row of the block sees
  // are left out.
  __device__ int chunks(int b) const {
    int64_t n = length(b);
    if (a.index) {
      n = n > 0 ? (int64_t)a.n_index << a.shift : 0;
    } else if (a.causal) {
      const int r0 = rb * rb_rows, r1 = min(r0 + rb_rows, a.heads_q / a.heads_kv * a.seqlen_q) - 1;
      const int last = r0 / a.seqlen_q == r1 / a.seqlen_q ? r1 % a.seqlen_q : a.seqlen_q - 1;
      n = n - a.seqlen_q + last + 1;
    }
    return (int)max((n + 31) >> 5, (int64_t)1);
  }
  // Every wave computes these alike, 64 sequences at a time.
  __device__ Shares shares(int lane, int least) const {
    Shares s;
    int sum = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) sum += b0 + lane < a.batch ? chunks(b0 + lane) : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    s.total = __builtin_amdgcn_readfirstlane(sum);
    s.count = min(a.shares, max(1, s.total / least));
    s.per = s.total / s.count;
    s.extra = s.total - s.per * s.count;
    return s;
  }
  // The sequence that holds chunk c, and the chunk it begins at.
  __device__ void find(int c, int lane, int& b, int& begin) const {
    int base = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      const int n = b0 + lane < a.batch ? chunks(b0 + lane) : 0;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(incl, o, 64);
        incl += lane >= o ? y : 0;
      }
      const int all = __builtin_amdgcn_readlane(incl, 63);
      if (base + all > c) {
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(base + incl > c));
        b = b0 + at;
        begin = base + __builtin_amdgcn_readlane(incl, at) - __builtin_amdgcn_readlane(n, at);
        return;
      }
      base += all;
    }
    b = a.batch;
    begin = base;
  }
};

// 16-bit value of the query's type.
__device__ inline uint16_t to_out(const PagedAttnArgs& a, float x) {
  return a.bf16 ? Elem<bf16_t>::from_f(x) : Elem<f16_t>::from_f(x);
}

// Merges the partials of one (sequence, head group, row block): those of
// workgroups j0 .. j1, the first of them in its second slot.
template <int D, int NT, bool AGENT>
__device__ inline void merge_partials(const PagedAttnArgs& a, int b, int hg, int rb, int nrb, int rb_rows, int j0, int j1,
                                      int tid) {
  const int hpw = 1 << a.head_shift, group = a.heads_q / a.heads_kv, rows = group * a.seqlen_q;
  const int here = min(rb_rows, rows - rb * rb_rows);
  auto ld = [](const float* p) {
    if constexpr (AGENT) return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else return *p;
  };
  for (int i = tid; i < hpw * here * D; i += NT) {
    const int d = i % D, r = (i / D) % here, hk = hg * hpw + i / (D * here);
    float M = kFloor, L = 0.f, o = 0.f;
    for (int j = j0; j <= j1; j += 8) {
      float m[8], l[8], x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int jj = min(j + u, j1);
        const int64_t row = (((int64_t)(2 * jj + (jj == j0 ? 1 : 0)) * a.heads_kv + hk) * nrb + rb) * rb_rows + r;
        m[u] = ld(a.ws_ml + 2 * row);
        l[u] = j + u <= j1 ? ld(a.ws_ml + 2 * row + 1) : 0.f;
        x[u] = ld(a.ws_o + row * D + d);
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < 8; ++u) top = fmaxf(top, m[u]);
      const float s = __builtin_amdgcn_exp2f(M - top);
      L *= s;
      o *= s;
      M = top;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = j + u <= j1 ? __builtin_amdgcn_exp2f(m[u] - top) : 0.f;
        L += w * l[u];
        if (j + u <= j1) o += w * x[u];
      }
    }
    const int row = rb * rb_rows + r, g = row / a.seqlen_q, q = row - g * a.seqlen_q;
    uint16_t* const op = reinterpret_cast<uint16_t*>(a.out) + b * a.out_stride[0] + (hk * group + g) * a.out_stride[1] +
                         q * a.out_stride[2];
    op[d] = to_out(a, L == 0.f ? 0.f : o / L);
  }
}

template <typename Tag, int KV, int D, int R, bool SMALL>
__global__ __launch_bounds__((AttnCfg<Tag, KV, D, R, SMALL>::NT)) void paged_attn_kernel(PagedAttnArgs a) {
  using C = AttnCfg<Tag, KV, D, R, SMALL>;
  using CT = typename std::conditional<C::KV8, f16_t, Tag>::type;  // type of the products
  using KE = typename std::conditional<C::KV8, uint8_t, uint16_t>::type;
  using KRaw = typename std::conditional<C::KREGS == 2, u32x2, u32x4>::type;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4, l16 = lane & 15;
  constexpr int RB = 16 * R;
  const int group = a.heads_q / a.heads_kv, rows = group * a.seqlen_q;
  const int nrb = (rows + RB - 1) / RB;
  const int rb_rows = min(RB, rows);
  const int hpw = 1 << a.head_shift, nhg = a.heads_kv >> a.head_shift;
  const int streams = C::NW >> a.head_shift;
  // KV heads fastest: neighbours in dispatch order read the same pages.
  const int hg = blockIdx.x % nhg, rb = blockIdx.x / nhg % nrb, share = blockIdx.x / (nhg * nrb);
  const int hw = wave & (hpw - 1), stream = wave >> a.head_shift;
  const int hk = hg * hpw + hw;
  const PagedWork work{a, rb_rows, rb};
  const Shares cut = work.shares(lane, 2 * streams);
  if (share >= cut.count) return;
  const int begin = cut.begin(share), end = cut.begin(share + 1);
  int b, b_begin;
  work.find(begin, lane, b, b_begin);

  const KE* const kbase = reinterpret_cast<const KE*>(a.k) + hk * a.k_stride[2];
  const KE* const vbase = reinterpret_cast<const KE*>(a.v) + hk * a.v_stride[2];
  uint16_t* const tile = reinterpret_cast<uint16_t*>(smem) + wave * (C::TILE_BYTES / 2);
  const int mask = (1 << a.shift) - 1;
  typedef const __attribute__((address_space(4))) int32_t const_i32;
  typedef const __attribute__((address_space(4))) float const_f32;

  for (int at = begin; at < end;) {
    const int len = work.length(b), all = work.chunks(b);
    const int c0 = at - b_begin, cnt = min(end, b_begin + all) - at;
    const int blocks = (len + mask) >> a.shift;           // logical blocks of the sequence
    const int listed = a.index ? a.n_index : blocks;
    const_i32* const index = (const_i32*)(a.index ? a.index + b * a.index_stride[0] + hk * a.index_stride[1] : nullptr);
    const_i32* const table = (const_i32*)(a.table + b * a.table_stride[0]);

    // --- Q ---------------------------------------------------------------
    s16x8 q[R][C::NSTEP];
    float qscale[R];
    int klim[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = rb * RB + 16 * r + l16;
      const bool valid = row < rows;
      const int g = valid ? row / a.seqlen_q : 0, m = valid ? row - g * a.seqlen_q : 0;
      klim[r] = a.causal ? len - a.seqlen_q + m : INT_MAX;
      const uint16_t* const src = reinterpret_cast<const uint16_t*>(a.q) + b * a.q_stride[0] +
                                  (hk * group + g) * a.q_stride[1] + m * a.q_stride[2];
#pragma unroll
      for (int s = 0; s < C::NSTEP; ++s) {
        // With paired K loads, lane group g4 covers 16 dims of a pair of steps.
        const int d = C::PAIR ? 64 * (s / 2) + 16 * g4 + 8 * (s % 2) : 32 * s + 8 * g4;
        q[r][s] = valid ? *reinterpret_cast<const s16x8*>(src + d) : zero_op<f16_t>();
      }
      qscale[r] = a.scale_log2;
      if (C::KV8 && a.bf16) {
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < C::NSTEP; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = fabsf(Elem<bf16_t>::to_f((uint16_t)q[r][s][e]));
            top = fmaxf(top, x < __builtin_inff() ? x : 0.f);
          }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const int ex = max((int)(__float_as_uint(top) >> 23), 15);
        const float down = __uint_as_float((uint32_t)(268 - ex) << 23);  // 2^(14 - (ex - 127))
        qscale[r] *= __uint_as_float((uint32_t)(ex - 14) << 23);
#pragma unroll
        for (int s = 0; s < C::NSTEP; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            q[r][s][e] = (short)Elem<f16_t>::from_f(Elem<bf16_t>::to_f((uint16_t)q[r][s][e]) * down);
      }
    }

    // --- what a chunk's keys are ------------------------------------------
    // Keys 16h .. 16h + 15 of a chunk (pages of 16 keys or more): one page.
    struct Half {
      int page, inside, key0, count;
      float ks, vs;
    };
    auto half_of = [&](int n) -> Half {
      Half h;
      const int at_list = n >> a.shift;
      bool ok = at_list < listed;
      int logical = at_list;
      if (a.index) {
        logical = index[(int64_t)min(at_list, listed - 1) * a.index_stride[2]];
        ok = ok && logical >= 0;
      }
      ok = ok && logical < blocks;
      const int page = table[(int64_t)min(max(logical, 0), a.max_blocks - 1) * a.table_stride[1]];
      ok = ok && page >= 0 && page < a.num_blocks;
      h.page = ok ? page : 0;
      h.inside = n & mask;
      h.key0 = ok ? (logical << a.shift) + h.inside : 0;
      h.count = ok ? min(max(len - h.key0, 0), 16) : 0;
      h.ks = h.vs = 1.f;
      if constexpr (C::KV8) {
        if (a.ks) h.ks = ((const_f32*)a.ks)[h.page * a.ks_stride[0] + hk * a.ks_stride[1]];
        if (a.vs) h.vs = ((const_f32*)a.vs)[h.page * a.vs_stride[0] + hk * a.vs_stride[1]];
      }
      h.vs = h.count ? h.vs : 0.f;
      return h;
    };
    // Pages of fewer keys: lane l describes key l % 32.
    struct Key {
      int64_t k, v;
      int pos, ok;
      float ks, vs;
    };
    auto key_of = [&](int n) -> Key {
      Key e;
      const int at_list = n >> a.shift;
      bool ok = at_list < listed;
      int logical = at_list;
      if (a.index) {
        logical = a.index[b * a.index_stride[0] + hk * a.index_stride[1] + (int64_t)min(at_list, listed - 1) * a.index_stride[2]];
        ok = ok && logical >= 0;
      }
      ok = ok && logical < blocks;
      int page = a.table[b * a.table_stride[0] + (int64_t)min(max(logical, 0), a.max_blocks - 1) * a.table_stride[1]];
      ok = ok && page >= 0 && page < a.num_blocks;
      page = ok ? page : 0;
      e.pos = ok ? (logical << a.shift) + (n & mask) : 0;
      e.ok = ok && e.pos < len;
      e.k = page * a.k_stride[0] + (n & mask) * a.k_stride[1];
      e.v = page * a.v_stride[0] + (n & mask) * a.v_stride[1];
      e.ks = e.vs = 1.f;
      if constexpr (C::KV8) {
        if (a.ks) e.ks = a.ks[page * a.ks_stride[0] + hk * a.ks_stride[1]];
        if (a.vs) e.vs = a.vs[page * a.vs_stride[0] + hk * a.vs_stride[1]];
      }
      e.vs = e.ok ? e.vs : 0.f;
      return e;
    };
    struct Meta {
      uint32_t there;         // bit k: key k of the chunk is one of the sequence's
      int key0[2];
      float ks[2], vs[2];     // SMALL: of the lane's key, in [0]
      int64_t voff[SMALL ? 1 : 2];
    };
    KRaw kr[C::NBUF][2][C::KN];
    u32x4 vr[C::NBUF][C::VN];
    Meta meta[C::NBUF];

    auto load_v = [&](const Meta& m, u32x4 (&vd)[C::VN]) {
#pragma unroll
      for (int i = 0; i < C::VN; ++i) {
        const int piece = 64 * i + lane, row = piece / C::PPR, col = piece % C::PPR * C::EPP;
        int64_t off;
        if constexpr (SMALL) {
          const uint32_t lo = __shfl((uint32_t)m.voff[0], row, 64), hi = __shfl((uint32_t)(m.voff[0] >> 32), row, 64);
          off = (int64_t)(((uint64_t)hi << 32) | lo);
        } else {
          off = (row < 16 ? m.voff[0] : m.voff[1]) + (row & 15) * a.v_stride[1];
        }
        vd[i] = *reinterpret_cast<const u32x4*>(vbase + off + col);
      }
    };
    auto issue = [&](int c, KRaw (&kd)[2][C::KN], u32x4 (&vd)[C::VN], Meta& m) {
      int64_t koff[2];
      if constexpr (SMALL) {
        const Key e = key_of(32 * c + (lane & 31));
        m.there = (uint32_t)__builtin_amdgcn_ballot_w64(e.ok != 0);
        m.key0[0] = e.pos;
        m.ks[0] = e.ks;
        m.vs[0] = e.vs;
        m.voff[0] = e.v;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t lo = __shfl((uint32_t)e.k, 16 * h + l16, 64), hi = __shfl((uint32_t)(e.k >> 32), 16 * h + l16, 64);
          koff[h] = (int64_t)(((uint64_t)hi << 32) | lo);
        }
      } else {
        m.there = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Half e = half_of(32 * c + 16 * h);
          m.there |= (e.count ? 0xFFFFu >> (16 - e.count) : 0u) << (16 * h);
          m.key0[h] = e.key0;
          m.ks[h] = e.ks;
          m.vs[h] = e.vs;
          m.voff[h] = e.page * a.v_stride[0] + e.inside * a.v_stride[1];
          koff[h] = e.page * a.k_stride[0] + (e.inside + l16) * a.k_stride[1];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int s = 0; s < C::KN; ++s) {
          const int d = C::PAIR ? 64 * s + 16 * g4 : 32 * s + 8 * g4;
          kd[h][s] = *reinterpret_cast<const KRaw*>(kbase + koff[h] + d);
        }
      if constexpr (!C::VLATE) load_v(m, vd);
    };

    // --- state -----------------------------------------------------------
    float m_i[R], l_i[R];
    f32x4a acc[R][C::NDB];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m_i[r] = kFloor;
      l_i[r] = 0.f;
#pragma unroll
      for (int i = 0; i < C::NDB; ++i) acc[r][i] = f32x4a{0.f, 0.f, 0.f, 0.f};
    }
    uint32_t vref = 0x00800000u;  // bits of a power of two

    auto compute = [&](const KRaw (&kd)[2][C::KN], const u32x4 (&vd)[C::VN], const Meta& m) {
      const bool whole = m.there == 0xFFFFFFFFu;
      // V to the tile; rows that are no keys as zeros (0 * NaN would be NaN).
      // `part`, see below: 0 all values; 1 finite ones, others 0; 2 a one for
      // each +inf or NaN; 3 a one for each -inf or NaN.
      auto piece_of = [&](int i) {
        const int row = (64 * i + lane) / C::PPR;
        u32x4 x = vd[i];
        if (!whole && !((m.there >> row) & 1u)) x = u32x4{0, 0, 0, 0};
        return x;
      };
      auto part_of = [&](s16x8 x, int part) {
        constexpr uint16_t EXP = std::is_same<CT, bf16_t>::value ? 0x7F80 : 0x7C00;
        const short one = (short)Elem<CT>::from_f(1.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint16_t u = (uint16_t)x[e];
          const bool odd = (u & EXP) == EXP, nan = (u & 0x7FFF) > EXP;
          const bool hit = odd && (nan || (u >> 15) == (part == 3));
          x[e] = part == 1 ? (odd ? (short)0 : x[e]) : hit ? one : (short)0;
        }
        return x;
      };
      auto fill = [&](int part) {
#pragma unroll
        for (int i = 0; i < C::VN; ++i) {
          const int piece = 64 * i + lane, row = piece / C::PPR, col = piece % C::PPR * C::EPP;
          const u32x4 x = piece_of(i);
          if constexpr (C::KV8) {
            s16x8 lo = codes_to_f16<KV>(u32x2{x[0], x[1]}), hi = codes_to_f16<KV>(u32x2{x[2], x[3]});
            if (part) { lo = part_of(lo, part); hi = part_of(hi, part); }
            *reinterpret_cast<s16x8*>(tile + swz_off<D>(row, col)) = lo;
            *reinterpret_cast<s16x8*>(tile + swz_off<D>(row, col + 8)) = hi;
          } else {
            s16x8 y = __builtin_bit_cast(s16x8, x);
            if (part) y = part_of(y, part);
            *reinterpret_cast<s16x8*>(tile + swz_off<D>(row, col)) = y;
          }
        }
      };
      fill(0);
      f32x4a s[R][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][h] = f32x4a{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < C::NSTEP; ++t) {
          s16x8 k;
          if constexpr (C::PAIR) {
            const u32x4 w = __builtin_bit_cast(u32x4, kd[h][t / 2]);
            k = codes_to_f16<KV>(t % 2 ? u32x2{w[2], w[3]} : u32x2{w[0], w[1]});
          } else if constexpr (C::KV8) {
            k = codes_to_f16<KV>(__builtin_bit_cast(u32x2, kd[h][t]));
          } else {
            k = __builtin_bit_cast(s16x8, kd[h][t]);
          }
#pragma unroll
          for (int r = 0; r < R; ++r) s[r][h] = mma16x16<CT>(k, q[r][t], s[r][h]);
        }
      }
      // Per key: scales (uniform over a half, or the key's own) and position.
      float ks[2][SMALL ? 4 : 1], w[2][SMALL ? 4 : 1];
      int pos[2][SMALL ? 4 : 1];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (SMALL) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = 16 * h + 4 * g4 + i;
            ks[h][i] = __shfl(m.ks[0], key, 64);
            w[h][i] = __shfl(m.vs[0], key, 64);
            pos[h][i] = __shfl(m.key0[0], key, 64);
          }
        } else {
          ks[h][0] = m.ks[h];
          w[h][0] = m.vs[h];
          pos[h][0] = m.key0[h] + 4 * g4;
        }
      }
      if constexpr (C::KV8) {
        uint32_t top;
        if constexpr (SMALL) {
          top = __float_as_uint(m.vs[0]) & 0x7FFFFFFFu;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        } else {
          top = max(__float_as_uint(m.vs[0]) & 0x7FFFFFFFu, __float_as_uint(m.vs[1]) & 0x7FFFFFFFu);
        }
        top = __builtin_amdgcn_readfirstlane(top);
        if (top > vref) {
          const uint32_t now = min((top + 0x7FFFFFu) & 0x7F800000u, 0x7E800000u);
          const float f = __uint_as_float((uint32_t)max((int)(0x3F800000u + vref - now), 0));
          vref = now;
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < C::NDB; ++i) acc[r][i] *= f;
        }
        const float inv = __uint_as_float(0x7F000000u - vref);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < (SMALL ? 4 : 1); ++i) w[h][i] *= inv;
      }
      // Some rows see keys of the chunk that others do not.
      bool mixed = a.causal && a.seqlen_q > 1;
      if constexpr (!SMALL) mixed = mixed && max(m.key0[0], m.key0[1]) + 15 > len - a.seqlen_q;
      const bool masked = SMALL || !whole || mixed;
      s16x8 p[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[r][h][i] *= qscale[r] * ks[h][SMALL ? i : 0];
        if (masked) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool seen = ((m.there >> (16 * h + 4 * g4 + i)) & 1u) && pos[h][SMALL ? i : 0] + (SMALL ? 0 : i) <= klim[r];
              s[r][h][i] = seen ? s[r][h][i] : kNegInf;
            }
        }
        float top = kNegInf;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, s[r][h][i]);
        if (__builtin_amdgcn_ballot_w64(top - m_i[r] > 8.f)) {
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float now = fmaxf(m_i[r], top), f = __builtin_amdgcn_exp2f(m_i[r] - now);
          m_i[r] = now;
          l_i[r] *= f;
#pragma unroll
          for (int i = 0; i < C::NDB; ++i) acc[r][i] *= f;
        }
        uint16_t e[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = __builtin_amdgcn_exp2f(s[r][h][i] - m_i[r]);
            l_i[r] += x;
            float y = C::KV8 ? x * w[h][SMALL ? i : 0] : x;
            if (masked) y = s[r][h][i] == kNegInf ? 0.f : y;  // (0 * a scale that is not finite)
            e[4 * h + i] = Elem<CT>::from_f(y);
          }
#pragma unroll
        for (int i = 0; i < 8; ++i) p[r][i] = (short)e[i];
      }
      const int trow = 4 * g4 + (l16 >> 2);
      typedef __attribute__((address_space(3))) s4a lds_s4;
      auto v_op = [&](int i) -> s16x8 {
        uint16_t* const t = tile + swz_off<D>(trow, 16 * i + 4 * (lane & 3));
        const s4a lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)t);
        const s4a hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(t + 16 * D));
        return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      };
      // A value that is not finite must not reach the rows that do not see
      // its key as 0 * inf: such a chunk takes the finite values first, then
      // adds an infinity wherever a row sees one.
      if constexpr (KV != FA_KV_INT8) {
        if (mixed) {
          uint32_t odd = 0;
#pragma unroll
          for (int i = 0; i < C::VN; ++i) {
            const u32x4 x = piece_of(i);
            constexpr uint32_t ABS = C::KV8 ? 0x7F7F7F7Fu : 0x7FFF7FFFu;
            constexpr uint32_t UP = C::KV8 ? 0x01010101u : std::is_same<CT, bf16_t>::value ? 0x00800080u : 0x04000400u;
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= ((x[e] & ABS) + UP) & ~ABS;
          }
          if (__builtin_amdgcn_ballot_w64(odd != 0)) {
            for (int part = 1; part < 4; ++part) {
              fill(part);
#pragma unroll
              for (int r = 0; r < R; ++r) {
                s16x8 ones;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  ones[e] = s[r][e / 4][e % 4] == kNegInf ? (short)0 : (short)Elem<CT>::from_f(1.f);
#pragma unroll
                for (int i = 0; i < C::NDB; ++i) {
                  const s16x8 v = v_op(i);
                  if (part == 1) {
                    acc[r][i] = mma16x16<CT>(v, p[r], acc[r][i]);
                  } else {
                    const f32x4a n = mma16x16<CT>(v, ones, f32x4a{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[r][i][e] += n[e] > 0.f ? (part == 2 ? -kNegInf : kNegInf) : 0.f;
                  }
                }
              }
            }
            return;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < C::NDB; ++i) {
        const s16x8 v = v_op(i);
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][i] = mma16x16<CT>(v, p[r], acc[r][i]);
      }
    };

    // --- the stream --------------------------------------------------------
    const int mine = cnt > stream ? (cnt - stream + streams - 1) / streams : 0;
    const int rounds = (mine + C::NBUF - 1) / C::NBUF;
    auto step = [&](int j) {
      if constexpr (C::VLATE) load_v(meta[j], vr[j]);
      compute(kr[j], vr[j], meta[j]);
    };
#pragma unroll
    for (int j = 0; j < C::NBUF; ++j) issue(c0 + stream + streams * j, kr[j], vr[j], meta[j]);
    for (int g = 0; g + 1 < rounds; ++g) {
#pragma unroll
      for (int j = 0; j < C::NBUF; ++j) {
        step(j);
        issue(c0 + stream + streams * ((g + 1) * C::NBUF + j), kr[j], vr[j], meta[j]);
      }
    }
    if (rounds > 0) {
#pragma unroll
      for (int j = 0; j < C::NBUF; ++j)
        if ((rounds - 1) * C::NBUF + j < mine) step(j);
    }

    // --- the waves of a head -------------------------------------------------
    const float vscale = C::KV8 ? __uint_as_float(vref) : 1.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l_i[r] += __shfl_xor(l_i[r], 16, 64);
      l_i[r] += __shfl_xor(l_i[r], 32, 64);
      if constexpr (C::KV8) {
#pragma unroll
        for (int i = 0; i < C::NDB; ++i) acc[r][i] *= vscale;
      }
    }
    float* const states = reinterpret_cast<float*>(smem);
    __syncthreads();
    for (int half = streams >> 1; half > 0; half >>= 1) {
      if (stream >= half && stream < 2 * half) {
        float* const st = states + (int64_t)((stream - half) * hpw + hw) * R * C::STATE * 64 + lane;
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int i = 0; i < C::NDB; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) st[(r * C::STATE + 4 * i + e) * 64] = acc[r][i][e];
          st[(r * C::STATE + 4 * C::NDB) * 64] = m_i[r];
          st[(r * C::STATE + 4 * C::NDB + 1) * 64] = l_i[r];
        }
      }
      __syncthreads();
      if (stream < half) {
        const float* const st = states + (int64_t)(stream * hpw + hw) * R * C::STATE * 64 + lane;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float m2 = st[(r * C::STATE + 4 * C::NDB) * 64], l2 = st[(r * C::STATE + 4 * C::NDB + 1) * 64];
          const float now = fmaxf(m_i[r], m2);
          const float f1 = __builtin_amdgcn_exp2f(m_i[r] - now), f2 = __builtin_amdgcn_exp2f(m2 - now);
          m_i[r] = now;
          l_i[r] = l_i[r] * f1 + l2 * f2;
#pragma unroll
          for (int i = 0; i < C::NDB; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[r][i][e] = acc[r][i][e] * f1 + st[(r * C::STATE + 4 * i + e) * 64] * f2;
        }
      }
      __syncthreads();
    }

    // --- out, or a partial -----------------------------------------------------
    const bool complete = cnt == all;
    if (stream == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int row = rb * RB + 16 * r + l16;
        if (row >= rows) continue;
        const int g = row / a.seqlen_q, mq = row - g * a.seqlen_q;
        if (complete) {
          const float inv = l_i[r] == 0.f ? 0.f : 1.f / l_i[r];
          uint16_t* const op = reinterpret_cast<uint16_t*>(a.out) + b * a.out_stride[0] +
                               (hk * group + g) * a.out_stride[1] + mq * a.out_stride[2] + 4 * g4;
#pragma unroll
          for (int i = 0; i < C::NDB; ++i) {
            s16x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (short)to_out(a, acc[r][i][e] * inv);
            *reinterpret_cast<s16x4*>(op + 16 * i) = o;
          }
        } else {
          const int64_t at_row = (((int64_t)(2 * share + (c0 == 0 ? 1 : 0)) * a.heads_kv + hk) * nrb + rb) * rb_rows +
                                 16 * r + l16;
          float* const po = a.ws_o + at_row * D + 4 * g4;
          float* const pm = a.ws_ml + 2 * at_row;
          if (a.tickets) {
            // Written through to where every XCD sees it (the L2s are not
            // coherent with each other).
#pragma unroll
            for (int i = 0; i < C::NDB; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                __hip_atomic_store(po + 16 * i + e, acc[r][i][e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (g4 == 0) {
              __hip_atomic_store(pm, m_i[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
              __hip_atomic_store(pm + 1, l_i[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
          } else {
#pragma unroll
            for (int i = 0; i < C::NDB; ++i) *reinterpret_cast<f32x4a*>(po + 16 * i) = acc[r][i];
            if (g4 == 0) {
              pm[0] = m_i[r];
              pm[1] = l_i[r];
            }
          }
        }
      }
    }
    if (!complete && a.tickets) {
      // The stores are acknowledged (vmcnt 0) before the workgroup's ticket;
      // no workgroup waits for another.
      int* const flag = reinterpret_cast<int*>(smem + C::LDS_BYTES - 16);
      wait_vm_all();
      __syncthreads();
      const int j0 = cut.owner(b_begin), j1 = cut.owner(b_begin + all - 1);
      if (tid == 0) {
        uint32_t* const t = a.tickets + ((int64_t)b * nhg + hg) * nrb + rb;
        const bool last = __hip_atomic_fetch_add(t, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(j1 - j0);
        if (last) __hip_atomic_store(t, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = last;
      }
      __syncthreads();
      const int last = *flag;
      if (last) merge_partials<D, C::NT, true>(a, b, hg, rb, nrb, rb_rows, j0, j1, tid);
      __syncthreads();
    }
    at += cnt;
    b_begin += all;
    ++b;
  }
}

// The merge as a launch of its own: grid (head groups * row blocks, batch).
template <typename Tag, int KV, int D, int R, bool SMALL>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs a) {
  using C = AttnCfg<Tag, KV, D, R, SMALL>;
  constexpr int RB = 16 * R;
  const int rows = a.heads_q / a.heads_kv * a.seqlen_q, nrb = (rows + RB - 1) / RB, rb_rows = min(RB, rows);
  const int nhg = a.heads_kv >> a.head_shift, hg = blockIdx.x % nhg, rb = blockIdx.x / nhg, lane = threadIdx.x & 63;
  const PagedWork work{a, rb_rows, rb};
  const Shares cut = work.shares(lane, 2 * (C::NW >> a.head_shift));
  int begin = 0;
  const int b = blockIdx.y;
  for (int b0 = 0; b0 < b; b0 += 64) begin += b0 + lane < b ? work.chunks(b0 + lane) : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) begin += __shfl_xor(begin, o, 64);
  const int j0 = cut.owner(begin), j1 = cut.owner(begin + work.chunks(b) - 1);
  if (j0 != j1) merge_partials<D, 256, false>(a, b, hg, rb, nrb, rb_rows, j0, j1, threadIdx.x);
}

}  // namespace fa
