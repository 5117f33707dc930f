// fa_paged_rows.hip - attention of many query rows (chunks of prompts) over a
// paged 8-bit cache with block scales: fa_paged_attn.hpp's shares and merge
// around a step that is bound by the matrix units, not by the stream.
//
// A workgroup has 128 packed query rows (head of the group, row), 32 a wave,
// and takes tiles of 64 keys that all four waves read: the codes are loaded
// and converted to fp16 once per workgroup, into one of two LDS buffers, while
// the other is in use (one barrier a tile).  S^T = K Q^T and O^T = V^T P^T with
// 32x32x16 products, so that P^T goes from its accumulators straight into the
// second one; V^T comes from the row-major tile transposed.  Two workgroups
// share a compute unit.  Scales, maxima, masks and values that are not finite
// are treated as in fa_paged_attn.hpp.  int8, 2 x 512 rows of 32/8 heads of 128
// over contexts up to 8192: 136 GFLOP in 186 us, 730 TFLOP/s (a large matrix
// product: 1190); the softmax of two waves a SIMD hides behind each other's
// products in part only.
#include "fa_paged_attn.hpp"

namespace fa {

template <int D>
struct RowsCfg {
  static constexpr int NW = 4, NT = 256, RB = kRowsBlock, KEYS = 64, UNIT = 6;
  static constexpr int STREAMS = 4;                // tiles a round counts for: a share has 8 at least
  static constexpr int NSTEP = D / 16, NDB = D / 32;
  static constexpr int PPR = D / 16;               // 16-code pieces of a row
  static constexpr int RPW = 64 / PPR;             // rows a wave loads at a time
  static constexpr int LOADS = KEYS / (NW * RPW);  // loads of a thread
  static constexpr int TILE = KEYS * D;            // elements
  static constexpr int LDS_BYTES = 2 * 2 * TILE * 2 + 16;
};

// (As in ShareRule, in rounds of four tiles.  int8, 32/8 heads of 128: 16 x 48 rows
// up to 900 keys 58.6 -> 52.3 us, up to 300 keys 59.5 -> 42; 8 x 200 rows up to 1500
// keys 110.5 -> 115.9, up to 2500 keys, with no limit, 123.5 -> 136.)
struct RowsShareRule {
  static constexpr int kPad = 2;
  static constexpr float kPadBelow = 4.f;
};

// PAGES: pages that a tile's 64 keys lie in (1, 2 or 4).
template <int KV, int D, int PAGES>
__global__ __launch_bounds__(256, 2) void paged_rows_kernel(PagedAttnArgs a) {
  using C = RowsCfg<D>;
  using EL = Elem<f16_t>;
  static_assert(KV != FA_KV_SAME, "8-bit caches");
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = a.heads_q / a.heads_kv, rows = group * a.seqlen_q;
  const SharePlace w(a, C::RB);
  const int hk = w.hg;
  const PagedWork work{a, w.rb_rows, w.rb, C::UNIT};
  const Shares cut = work.shares<RowsShareRule>(lane, C::STREAMS);
  if (w.share >= cut.count) return;
  const int begin = cut.begin(w.share), end = cut.begin(w.share + 1);
  int b, b_begin;
  work.find(begin, cut.pad, lane, b, b_begin);

  typedef const unsigned char* bytes;
  typedef const __attribute__((address_space(4))) int32_t const_i32;
  typedef const __attribute__((address_space(4))) float const_f32;
  const bytes kbase = static_cast<bytes>(a.k) + hk * a.k_stride[2], vbase = static_cast<bytes>(a.v) + hk * a.v_stride[2];
  const int prow = lane / C::PPR, pcol = lane % C::PPR;
  const int mask = (1 << a.shift) - 1;
  const uint32_t t1 = (uint32_t)a.table_stride[1];
  const float* const ks_head = a.ks ? a.ks + hk * a.ks_stride[1] : nullptr;
  const float* const vs_head = a.vs ? a.vs + hk * a.vs_stride[1] : nullptr;
  uint16_t* const tiles = reinterpret_cast<uint16_t*>(smem);
  int* const flag = reinterpret_cast<int*>(smem + C::LDS_BYTES - 16);  // values were left out
  constexpr int KEYS_PP = C::KEYS / PAGES;  // keys of a page's part

  for (int at = begin; at < end;) {
    const int len = work.length(b), all = work.chunks(b);
    b_begin += cut.pad;
    at = max(at, b_begin);
    const int c0 = at - b_begin, cnt = min(end, b_begin + all) - at;
    if (cnt <= 0) break;  // (the share ends before the sequence's first tile)
    const int blocks = (len + mask) >> a.shift;
    const int listed = a.index ? a.n_index : blocks;
    const int32_t* const index = a.index ? a.index + b * a.index_stride[0] + hk * a.index_stride[1] : nullptr;
    const_i32* const table = (const_i32*)(a.table + b * a.table_stride[0]);

    // A tile is known two steps ahead by its logical blocks, one step by its
    // pages, so that no scalar load is waited for at its place.
    struct Ahead {
      int logical[PAGES], page[PAGES];
    };
    auto logical_of = [&](int n) {  // of the listed block that holds key n of the list
      const int at_list = n >> a.shift;
      if (!index) return at_list;
      const int l = ((const_i32*)index)[(int64_t)min(at_list, listed - 1) * a.index_stride[2]];
      return at_list < listed ? l : -1;
    };
    auto page_of = [&](int logical) { return table[(uint64_t)(uint32_t)min(max(logical, 0), a.max_blocks - 1) * t1]; };
    struct Meta {
      int inside, page[PAGES], key0[PAGES], here[PAGES];  // here: keys from the part's first on (0: none)
      float ks[PAGES], vs[PAGES];
    };
    auto describe = [&](int t, const Ahead& x) -> Meta {
      Meta m;
      m.inside = (C::KEYS * t) & mask;
#pragma unroll
      for (int p = 0; p < PAGES; ++p) {
        const bool ok = (uint32_t)x.logical[p] < (uint32_t)blocks && (uint32_t)x.page[p] < (uint32_t)a.num_blocks;
        m.page[p] = ok ? x.page[p] : 0;
        m.key0[p] = (x.logical[p] << a.shift) + (PAGES == 1 ? m.inside : 0);
        m.here[p] = ok ? max(len - m.key0[p], 0) : 0;
        m.ks[p] = a.ks ? ((const_f32*)ks_head)[m.page[p] * a.ks_stride[0]] : 1.f;
        m.vs[p] = a.vs ? ((const_f32*)vs_head)[m.page[p] * a.vs_stride[0]] : 1.f;
        m.vs[p] = m.here[p] ? m.vs[p] : 0.f;
      }
      return m;
    };

    // --- this lane's query row --------------------------------------------
    const int row = w.rb * C::RB + 32 * wave + l32;
    const bool valid = row < rows;
    const int g = valid ? row / a.seqlen_q : 0, mq = valid ? row - g * a.seqlen_q : 0;
    const int lim = min(a.causal ? len - a.seqlen_q + mq : INT_MAX, len - 1);  // last key it sees
    s16x8 q[C::NSTEP];
    {
      const uint16_t* const src = reinterpret_cast<const uint16_t*>(a.q) + b * a.q_stride[0] +
                                  (hk * group + g) * a.q_stride[1] + mq * a.q_stride[2] + 8 * h;
#pragma unroll
      for (int s = 0; s < C::NSTEP; ++s) q[s] = valid ? *reinterpret_cast<const s16x8*>(src + 16 * s) : zero_op<f16_t>();
    }
    float qscale = a.scale_log2;
    if (a.bf16) qscale *= bf16_row_to_f16(q, half_max(bf16_row_top(q)));
    float zero = 0.f;
    if constexpr (KV == FA_KV_INT8) {
      const short c = (short)EL::from_f(-kInt8Offset);
      const s16x8 off = {c, c, c, c, c, c, c, c};
      f32x16 x = zero16();
#pragma unroll
      for (int s = 0; s < C::NSTEP; ++s) x = EL::mma(off, q[s], x);
      zero = x[0];
    }

    // --- staging: the wave's rows of a tile, registers -> LDS ---------------
    u32x4 kd[C::LOADS], vd[C::LOADS];
    int vhere[C::LOADS], vkey[C::LOADS];  // keys from this thread's row on, and its position
    auto load = [&](const Meta& m) {
#pragma unroll
      for (int i = 0; i < C::LOADS; ++i) {
        // A wave's rows of one load lie in one page (RPW <= 16).
        const int first = (i * C::NW + wave) * C::RPW, p = first / KEYS_PP, in = first - p * KEYS_PP;
        int page = m.page[0], key0 = m.key0[0], here = m.here[0];
#pragma unroll
        for (int x = 1; x < PAGES; ++x) {
          page = p == x ? m.page[x] : page;
          key0 = p == x ? m.key0[x] : key0;
          here = p == x ? m.here[x] : here;
        }
        const int64_t inside = (PAGES == 1 ? m.inside : 0) + in + prow;
        kd[i] = *reinterpret_cast<const u32x4*>(kbase + page * a.k_stride[0] + inside * a.k_stride[1] + 16 * pcol);
        vd[i] = *reinterpret_cast<const u32x4*>(vbase + page * a.v_stride[0] + inside * a.v_stride[1] + 16 * pcol);
        vhere[i] = here - in - prow;
        vkey[i] = key0 + in + prow;
      }
    };
    auto stage = [&](int buf) {
      uint16_t* const kt = tiles + buf * 2 * C::TILE;
      uint16_t* const vt = kt + C::TILE;
#pragma unroll
      for (int i = 0; i < C::LOADS; ++i) {
        const int r = (i * C::NW + wave) * C::RPW + prow;
        u32x4 x = vd[i];
        if (vhere[i] <= 0) x = u32x4{0, 0, 0, 0};  // (0 * NaN would be NaN)
        if constexpr (KV != FA_KV_INT8) {
          // Values that are not finite, of keys that some row does not see.
          if (a.causal && a.seqlen_q > 1 && vkey[i] > len - a.seqlen_q) {
            uint32_t odd = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t bad = ((x[e] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
              x[e] &= ~((bad >> 7) * 0xFFu);
              odd |= bad;
            }
            if (odd) *flag = 1;
          }
        }
        *reinterpret_cast<s16x8*>(kt + swz_off<D>(r, 16 * pcol)) = codes_to_f16<KV, true>(u32x2{kd[i][0], kd[i][1]});
        *reinterpret_cast<s16x8*>(kt + swz_off<D>(r, 16 * pcol + 8)) = codes_to_f16<KV, true>(u32x2{kd[i][2], kd[i][3]});
        *reinterpret_cast<s16x8*>(vt + swz_off<D>(r, 16 * pcol)) = codes_to_f16<KV, false>(u32x2{x[0], x[1]});
        *reinterpret_cast<s16x8*>(vt + swz_off<D>(r, 16 * pcol + 8)) = codes_to_f16<KV, false>(u32x2{x[2], x[3]});
      }
    };
    // Before a row has seen a key its maximum counts as 0 and its sums are 0.
    float m_i = 0.f, l_i = 0.f;
    bool fresh = true;
    f32x16 acc[C::NDB];
#pragma unroll
    for (int i = 0; i < C::NDB; ++i) acc[i] = zero16();
    uint32_t vref = 0x00800000u;

    auto compute = [&](int buf, const Meta& m) {
      const uint16_t* const kt = tiles + buf * 2 * C::TILE;
      const uint16_t* const vt = kt + C::TILE;
      uint32_t scale_top = 0;
      bool masked = false;
#pragma unroll
      for (int p = 0; p < PAGES; ++p) {
        scale_top = max(scale_top, __float_as_uint(m.vs[p]) & 0x7FFFFFFFu);
        masked = masked || m.here[p] < KEYS_PP || (a.causal && m.key0[p] + KEYS_PP - 1 > len - a.seqlen_q);
      }
      scale_top = __builtin_amdgcn_readfirstlane(scale_top);
      if (scale_top > vref) {
        const uint32_t grown = min((scale_top + 0x7FFFFFu) & 0x7F800000u, 0x7E800000u);
        const float f = __uint_as_float((uint32_t)max((int)(0x3F800000u + vref - grown), 0));
        vref = grown;
#pragma unroll
        for (int i = 0; i < C::NDB; ++i) acc[i] *= f;
      }
      const bool odd_scale = scale_top >= 0x7F800000u;
      const float inv = __uint_as_float(0x7F000000u - vref);
      float f[PAGES], wv[PAGES];
#pragma unroll
      for (int p = 0; p < PAGES; ++p) {
        f[p] = qscale * m.ks[p];
        wv[p] = m.vs[p] * inv;
      }
      // Blocks of 32 keys, one after the other (both at once: 30 registers too many).
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        f32x16 x;  // the sums, then the logits relative to the maximum
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = zero;
#pragma unroll
        for (int t = 0; t < C::NSTEP; ++t)
          x = EL::mma(*reinterpret_cast<const s16x8*>(kt + swz_off<D>(32 * kb + l32, 16 * t + 8 * h)), q[t], x);
        // Element i: key 32 kb + acc_row(i, h), in this part of the tile.
        auto part = [&](int i) { return (32 * kb + 8 * (i >> 2)) / KEYS_PP; };
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(x[i], f[part(i)], -m_i);
        if (masked) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int p = part(i), key = 32 * kb + 8 * (i >> 2) + (i & 3) - KEYS_PP * p + 4 * h;
            x[i] = m.here[p] > 0 && m.key0[p] + key <= lim ? x[i] : kNegInf;
          }
        }
        float top = kNegInf;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, x[i]);
        top = half_max(top);
        const bool some = top > kNegInf;
        if (__builtin_amdgcn_ballot_w64(top > 8.f || (fresh && some && top < -8.f))) {
          const float up = fresh ? (some ? top : 0.f) : fmaxf(top, 0.f);
          const float down = fresh ? 1.f : __builtin_amdgcn_exp2f(-up);
          m_i += up;
          l_i *= down;
#pragma unroll
          for (int i = 0; i < C::NDB; ++i) acc[i] *= down;
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] -= up;
        }
        fresh = fresh && !some;
        s16x8 p[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int i = 8 * j + e;
            const float y = __builtin_amdgcn_exp2f(x[i]);
            l_i += y;
            float z = y * wv[part(i)];
            if (__builtin_expect(odd_scale, 0)) z = x[i] == kNegInf ? 0.f : z;
            p[j][e] = (short)EL::from_f(z);
          }
#pragma unroll
        for (int db = 0; db < C::NDB; ++db)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[db] = EL::mma(tr_op_rowmap<D>(vt, 0, 32 * db, 2 * kb + j, lane), p[j], acc[db]);
      }
    };

    // --- the tiles -----------------------------------------------------------
    if (tid == 0) *flag = 0;
    auto tile = [&](int t) { return min(c0 + t, c0 + cnt - 1); };
    Ahead first, next;
    int later[PAGES];
#pragma unroll
    for (int p = 0; p < PAGES; ++p) {
      first.logical[p] = logical_of(C::KEYS * tile(0) + KEYS_PP * p);
      next.logical[p] = logical_of(C::KEYS * tile(1) + KEYS_PP * p);
      later[p] = logical_of(C::KEYS * tile(2) + KEYS_PP * p);
    }
#pragma unroll
    for (int p = 0; p < PAGES; ++p) {
      first.page[p] = page_of(first.logical[p]);
      next.page[p] = page_of(next.logical[p]);
    }
    Meta now = describe(tile(0), first);
    load(now);
    __syncthreads();  // the last sequence's tiles are read, the flag is clear
    stage(0);
    __syncthreads();
#pragma unroll 1
    for (int t = 0; t < cnt; ++t) {
      const bool more = t + 1 < cnt;
      const Meta m = now;
      if (more) {
        now = describe(tile(t + 1), next);
        load(now);
#pragma unroll
        for (int p = 0; p < PAGES; ++p) {
          next.logical[p] = later[p];
          next.page[p] = page_of(later[p]);
          later[p] = logical_of(C::KEYS * tile(t + 3) + KEYS_PP * p);
        }
      }
      compute(t & 1, m);
      if (more) stage((t + 1) & 1);
      __syncthreads();
    }
    const bool left_out = *flag != 0;
    __syncthreads();  // (the next sequence clears the flag)
    if (KV != FA_KV_INT8 && __builtin_expect(left_out, 0)) {
      // The values that were left out, key by key.
#pragma unroll 1
      for (int k = max(C::KEYS * c0, 0); k < C::KEYS * (c0 + cnt); ++k) {
        const int logical = logical_of(k), page = page_of(logical), key = (logical << a.shift) + (k & mask);
        if ((uint32_t)logical >= (uint32_t)blocks || (uint32_t)page >= (uint32_t)a.num_blocks || key >= len ||
            key <= len - a.seqlen_q)
          continue;
        const float vs = a.vs ? vs_head[page * a.vs_stride[0]] : 1.f;
        const bytes at_v = vbase + page * a.v_stride[0] + (k & mask) * a.v_stride[1];
#pragma unroll
        for (int db = 0; db < C::NDB; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if ((at_v[32 * db + acc_row(i, h)] & 0x7F) == 0x7F && key <= lim) acc[db][i] += __builtin_nanf("") * vs;
      }
    }

    // --- out, or a partial -----------------------------------------------------
    l_i = half_sum(l_i);
    m_i = fresh ? kFloor : m_i;
    const float vscale = __uint_as_float(vref);
    const bool complete = cnt == all;
    if (valid) {
      const float inv = complete ? (l_i == 0.f ? 0.f : vscale / l_i) : vscale;
      const int64_t part = partial_row(a, 2 * w.share + (c0 == 0 ? 1 : 0), hk, w.rb, w.nrb, w.rb_rows) + 32 * wave + l32;
#pragma unroll
      for (int db = 0; db < C::NDB; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const f32x4a o = {acc[db][i] * inv, acc[db][i + 1] * inv, acc[db][i + 2] * inv, acc[db][i + 3] * inv};
          const int d = 32 * db + acc_row(i, h);
          if (complete) store_out(a, b, hk, row, d, o);
          else *reinterpret_cast<f32x4a*>(a.ws_o + part * D + d) = o;
        }
      if (!complete && h == 0) {
        a.ws_ml[2 * part] = m_i;
        a.ws_ml[2 * part + 1] = l_i;
      }
    }
    at += cnt;
    b_begin += all;
    ++b;
  }
}

namespace {

template <int KV, int D, int PAGES>
hipError_t run_rows(const PagedAttnArgs& a, int nrb, hipStream_t stream) {
  using C = RowsCfg<D>;
  auto kern = paged_rows_kernel<KV, D, PAGES>;
  hipError_t e = allow_lds((const void*)kern, C::LDS_BYTES);
  if (e != hipSuccess) return e;
  const int columns = a.heads_kv * nrb;
  hipLaunchKernelGGL(kern, dim3((unsigned)(columns * a.shares)), dim3(C::NT), C::LDS_BYTES, stream, a);
  e = hipGetLastError();
  if (e != hipSuccess || a.shares == 1) return e;
  // A block's partials are 64 KiB a share: the last workgroup alone takes longer
  // to merge them than a second launch does (64 rows of 32 heads over 8192 keys,
  // 32 shares: 208 us in all against 48).
  const int rb_rows = std::min(C::RB, a.heads_q / a.heads_kv * a.seqlen_q);
  hipLaunchKernelGGL((paged_merge_kernel<D, C::RB, C::UNIT, C::STREAMS, RowsShareRule>),
                     dim3((unsigned)columns, (unsigned)a.batch, (unsigned)((rb_rows * (D / 4) + 255) / 256)), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

template <int KV, int D>
hipError_t run_pages(const PagedAttnArgs& a, int nrb, hipStream_t s) {
  if (a.shift >= 6) return run_rows<KV, D, 1>(a, nrb, s);
  if (a.shift == 5) return run_rows<KV, D, 2>(a, nrb, s);
  return run_rows<KV, D, 4>(a, nrb, s);
}

}  // namespace

hipError_t launch_paged_rows(const PagedAttnArgs& a, int kv_format, int head_dim, int nrb, hipStream_t s) {
  const bool e4m3 = kv_format == FA_KV_E4M3;
  switch (head_dim) {
    case 64: return e4m3 ? run_pages<FA_KV_E4M3, 64>(a, nrb, s) : run_pages<FA_KV_INT8, 64>(a, nrb, s);
    case 128: return e4m3 ? run_pages<FA_KV_E4M3, 128>(a, nrb, s) : run_pages<FA_KV_INT8, 128>(a, nrb, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace fa
