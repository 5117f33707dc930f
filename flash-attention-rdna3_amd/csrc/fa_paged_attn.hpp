// fa_paged_attn.hpp - attention over a paged cache whose codes have a scale for
// each block and head, over all blocks of a sequence or over listed ones.
//
//   S_rj = softmax_scale * ks[page(j)] * (q_r . k_j),   O_r = sum_j p_rj vs[page(j)] v_j / sum_j p_rj,
//   p_rj = exp(S_rj - m_r)
//
// One pass over the keys with a running maximum and sum, fp32 throughout.
//
//  * Work.  The keys of all sequences are one line of 32-key chunks, cut into
//    equal shares, one for each workgroup of a (head group, row block): no
//    workgroup has more than another, whatever the lengths.  A share holds the
//    end of one sequence, whole ones, and the start of another; sequences that
//    several shares hold are merged from unnormalised partials by the last
//    workgroup that arrives (or by a second launch).
//  * Stream.  A wave has one chunk in registers, whole rows of K and of V as
//    16-byte pieces (whole cache lines an instruction; loads in the matrix
//    instruction's own layout take 64 bytes of a row each and measured 4 %
//    slower).  It writes them to LDS tiles of its own, asks for its next chunk
//    at once, and reads K back by rows and V transposed.  Page ids and scales
//    are scalar loads a chunk or two ahead, so that they do not wait behind
//    the stream.  A second chunk in registers measured 6 % slower.
//  * Heads.  A workgroup takes as many KV heads as fill 256 bytes of a token's
//    row, its waves shared out among them (int8, contexts up to 131072: 179 us
//    with one head of 128 bytes, 166 with two, 166 with four).
//  * Types.  8-bit codes are fp16 numbers exactly, so over 8-bit caches the
//    products run in fp16 whatever the query's type: a bfloat16 query row is
//    scaled by a power of two to a largest value of 2^14 first (its 8 bits fit;
//    what is 2^-28 of the row's largest value loses bits).  ks joins the logit
//    scale.  p is rounded to fp16 with vs / vref on it, vref the largest power
//    of two seen over the scales: at most 2^8, and relative to what dominates.
//  * The sum of the weights takes each p as it was rounded, so that a row of few
//    keys does not carry the rounding twice (vs / vref below 2^-5: as it was,
//    for there the rounded one may have lost its bits).  It costs nothing here,
//    36.1 us either way over 134 MB of e4m3; in the kernel of many query rows,
//    which is bound by its instructions, 225 us against 204: there l sums p.
//  * What bounds it: the stream.  int8, 4 contexts up to 131072 of 8 heads of 128,
//    854 MB: 152 us, 5.6 TB/s (a read alone: 7.0); e4m3, 4 x 16384, 134 MB: 35 us,
//    of which ramp, first chain of loads and merge are some 10.
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
  int64_t k_stride[3];  // block, position, head; in bytes
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
  int32_t head_shift;    // log2 of the KV heads of a group: a workgroup's waves share them out
  float* ws_o;           // [2 * shares][heads_kv][row blocks][rows of a block][D]
  float* ws_ml;          // the same without D, pairs (m, l)
  uint32_t* tickets;
};

// The kernel for many query rows (fa_paged_rows.hip): 8-bit caches, head dim 64
// or 128, pages of 16 keys or more; a.shares workgroups for each KV head and
// each of `nrb` blocks of kRowsBlock rows.
constexpr int kRowsBlock = 128;
hipError_t launch_paged_rows(const PagedAttnArgs& a, int kv_format, int head_dim, int nrb, hipStream_t stream);

// How a chunk finds its pages.  Strides below 2^31 bytes, one page for its 32
// keys or one for each half: scalar loads and 32-bit products.  Else each lane
// finds the page of a key of its own.
enum PageMode { kOnePage, kTwoPages, kAnyPages };

template <typename Tag, int KV, int D, int PAGES>
struct AttnCfg {
  static constexpr bool KV8 = KV != FA_KV_SAME;
  static constexpr int ES = KV8 ? 1 : 2;                      // bytes of an element
  static constexpr int PPR = D * ES / 16;                     // 16-byte pieces of a row
  static constexpr int VN = 32 * PPR / 64;                    // loads of 32 rows
  static constexpr int TILE = 32 * D * ES;                    // bytes of one operand's tile
  // Waves: two per SIMD where their registers and tiles have room.
  static constexpr int NW = TILE >= 32768 ? 2 : TILE >= 16384 ? 4 : 8;
  static constexpr int NT = 64 * NW;
  static constexpr int RB = 16;                               // rows of a row block
  static constexpr int NSTEP = D / 32;                        // 32-dim steps of Q K^T
  static constexpr int NDB = D / 16;                          // 16-dim blocks of O
  static constexpr bool PAIR = KV8 && NSTEP > 1;              // 16 bytes of K serve two steps
  // Rows of 128 bytes and more are whole cache lines of one head, read once.
  static constexpr bool ONCE = D * ES >= 128;
  static constexpr int LOOP_BYTES = 2 * NW * TILE;
  static constexpr int OLD = D + 4;                           // row stride of the waves' sums (floats)
  static constexpr int MERGE_BYTES = NW * RB * (OLD + 2) * 4;
  static constexpr int LDS_BYTES = (LOOP_BYTES > MERGE_BYTES ? LOOP_BYTES : MERGE_BYTES) + 16;  // + ticket flag
};

template <typename Tag> __device__ inline f32x4a mma16x16(s16x8 a, s16x8 b, f32x4a c);
template <> __device__ inline f32x4a mma16x16<f16_t>(s16x8 a, s16x8 b, f32x4a c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
}
template <> __device__ inline f32x4a mma16x16<bf16_t>(s16x8 a, s16x8 b, f32x4a c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}

// int8 codes x as fp16 1152 + x (bits 0x6400 + 128 + x).  In Q K^T the 1152
// times the row's sum is taken off by the accumulator's first value: the sums
// then pass through values of up to ten times those of |q| |k|, in fp32 still
// 2^-20 of them.  (Not for V, where the sum runs over all the keys.)
constexpr float kInt8Offset = 1152.f;
template <bool OFFSET>
__device__ inline s16x8 int8x8_to_f16(u32x2 r) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = r[i / 2] ^ 0x80808080u;
    o[i] = __builtin_amdgcn_perm(0x64646464u, u, i % 2 ? 0x04030402u : 0x04010400u);
    if constexpr (!OFFSET) {
      const h16x2 c = {(_Float16)kInt8Offset, (_Float16)kInt8Offset};
      const h16x2 x = __builtin_bit_cast(h16x2, o[i]) - c;
      o[i] = __builtin_bit_cast(uint32_t, x);
    }
  }
  return __builtin_bit_cast(s16x8, u32x4{o[0], o[1], o[2], o[3]});
}

// Eight codes as fp16, exactly; for K, int8 ones with the offset.
template <int KV, bool K> __device__ inline s16x8 codes_to_f16(u32x2 r) {
  if constexpr (KV == FA_KV_INT8) return int8x8_to_f16<K>(r);
  else return fp8x8_to_op<f16_t>(r);
}

// Byte offset of 16-byte piece c of row r in a tile of rows of N pieces: the
// pieces of the rows that an access touches together lie in different banks.
template <int N> __device__ constexpr inline int piece_off(int r, int c) {
  constexpr int PER = N >= 8 ? 1 : 8 / N;  // rows of 128 bytes
  return (r * N + (c ^ (r / PER & (N >= 8 ? 7 : N - 1)))) * 16;
}

constexpr float kFloor = -3.0e38f;  // the running maximum before any key

// How the chunks of a (head group, row block) are shared out: `total` chunks
// over `count` workgroups, the first `extra` of them with one more.  `pad` of
// them are no work: they stand before each sequence's for what its beginning
// costs.
struct Shares {
  int total, count, per, extra, pad;
  __device__ int begin(int j) const { return j * per + min(j, extra); }
  __device__ int owner(int c) const {
    const int big = extra * (per + 1);
    return c < big ? c / (per + 1) : extra + (c - big) / per;
  }
};

// A sequence's first chunk waits for its length, table, page and rows in turn: as
// long as kPad rounds of a workgroup's streams take.  Counted where the sequences
// have fewer than kPadBelow rounds; longer ones gain nothing by it, and lose the
// cuts at their ends.  (e4m3, 32/8 heads of 128, 32 sequences up to 2000 keys: 30.5
// -> 23.1 us, 1 and 2 rounds 25.6 and 24.3; up to 64 x 1200: 40 -> 27.7; 16 lists of
// 64 blocks of 64, 32 rounds: 33.1, with it 35.2.)
struct ShareRule {
  static constexpr int kPad = 3;
  static constexpr float kPadBelow = 20.f;
};

struct PagedWork {
  const PagedAttnArgs& a;
  int rb_rows, rb;  // rows of a row block, and the row block
  int unit;         // log2 of a chunk's keys
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
    return (int)max((n + (1 << unit) - 1) >> unit, (int64_t)1);
  }
  // Every wave computes these alike, 64 sequences at a time.  A workgroup takes
  // `streams` chunks at a time, a power of two.
  template <typename RULE> __device__ Shares shares(int lane, int streams) const {
    Shares s;
    int sum = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) sum += b0 + lane < a.batch ? chunks(b0 + lane) : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    sum = __builtin_amdgcn_readfirstlane(sum);
    const float steps = (float)sum * __builtin_amdgcn_rcpf((float)(a.batch * streams));  // mean rounds of a sequence
    s.pad = steps < RULE::kPadBelow ? RULE::kPad * streams - 1 : 0;
    s.total = sum + s.pad * a.batch;
    s.count = max(1, min(a.shares, s.total >> __builtin_ctz(2 * streams)));
    // A sequence's partials are read one after the other, a share's rounds as well:
    // with fewer shares the one takes less, the other more.  (int8, 3 sequences up to
    // 6486 keys of 8 heads of 32: 49 us without this limit, with the factor 1, 1.5
    // and 2 38, 34.3 and 33.5; 4 x 16384 e4m3, 8 heads of 128: 40.2 with 1, else 37.3.)
    s.count = min(s.count, (int)((float)a.batch * (1.f + 2.f * __builtin_amdgcn_sqrtf(steps))));
    s.per = s.total / s.count;
    s.extra = s.total - s.per * s.count;
    return s;
  }
  // The sequence that holds chunk c, and the chunk it begins at.
  __device__ void find(int c, int pad, int lane, int& b, int& begin) const {
    int base = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      const int n = b0 + lane < a.batch ? chunks(b0 + lane) + pad : 0;
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

// Four dims of an output row.
__device__ inline void store_out(const PagedAttnArgs& a, int b, int hk, int row, int d, const f32x4a& o) {
  const int group = a.heads_q / a.heads_kv, g = row / a.seqlen_q, m = row - g * a.seqlen_q;
  uint16_t* const op = reinterpret_cast<uint16_t*>(a.out) + b * a.out_stride[0] + (hk * group + g) * a.out_stride[1] +
                       m * a.out_stride[2] + d;
  s16x4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = (short)to_out(a, o[e]);
  *reinterpret_cast<s16x4*>(op) = x;
}

// Partials of shares that one launch merges are written through to where
// every XCD sees them and read from there (the XCDs' L2s are not coherent
// with each other): cache policy "agent scope".
constexpr int kAgent = 16;
__device__ inline __amdgpu_buffer_rsrc_t rsrc_of(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, 0x7FFFFFFF, 0x00020000);
}

// Index of a partial's row block: `slot` 2 * share, + 1 for the share's last
// sequence if it goes on behind the share.
__device__ inline int64_t partial_row(const PagedAttnArgs& a, int slot, int hk, int rb, int nrb, int rb_rows) {
  return (((int64_t)slot * a.heads_kv + hk) * nrb + rb) * rb_rows;
}

// Merges the partials of one (sequence, head group, row block): those of the
// workgroups j0 .. j1, the first of them in its second slot.
template <int D, bool AGENT>
__device__ inline void merge_partials(const PagedAttnArgs& a, int b, int hg, int rb, int nrb, int rb_rows, int j0, int j1,
                                      int tid, int threads) {
  const int rows = a.heads_q / a.heads_kv * a.seqlen_q, heads = 1 << a.head_shift;
  const int here = min(rb_rows, rows - rb * rb_rows);
  const __amdgpu_buffer_rsrc_t ro = rsrc_of(a.ws_o), rm = rsrc_of(a.ws_ml);
  typedef float f32x2a __attribute__((ext_vector_type(2)));
  for (int i = tid; i < heads * here * (D / 4); i += threads) {
    const int d = i % (D / 4) * 4, r = i / (D / 4) % here, hk = hg * heads + i / (D / 4 * here);
    float M = kFloor, L = 0.f;
    f32x4a o = {0.f, 0.f, 0.f, 0.f};
    for (int j = j0; j <= j1; j += 4) {
      f32x2a ml[4];
      f32x4a x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int jj = min(j + u, j1);
        const int64_t row = partial_row(a, 2 * jj + (jj == j0 ? 1 : 0), hk, rb, nrb, rb_rows) + r;
        if constexpr (AGENT) {
          // (bit_cast the whole result: subscripting the builtin's vector
          // directly compiles to one dword load splatted to all four.)
          ml[u] = __builtin_bit_cast(f32x2a, __builtin_amdgcn_raw_buffer_load_b64(rm, (int)(row * 8), 0, kAgent));
          x[u] = __builtin_bit_cast(f32x4a, __builtin_amdgcn_raw_buffer_load_b128(ro, (int)((row * D + d) * 4), 0, kAgent));
        } else {
          ml[u] = *reinterpret_cast<const f32x2a*>(a.ws_ml + 2 * row);
          x[u] = *reinterpret_cast<const f32x4a*>(a.ws_o + row * D + d);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (j + u > j1) break;
        const float top = fmaxf(M, ml[u][0]);
        const float s = __builtin_amdgcn_exp2f(M - top), w = __builtin_amdgcn_exp2f(ml[u][0] - top);
        L = L * s + ml[u][1] * w;
        o = o * s + x[u] * w;
        M = top;
      }
    }
    store_out(a, b, hk, rb * rb_rows + r, d, o * (L == 0.f ? 0.f : 1.f / L));
  }
}

// What the shares' kernels have in common: which share this is, and its place
// in the line of chunks.
struct SharePlace {
  int hg, rb, share, nrb, rb_rows;
  // Head groups fastest: neighbours in dispatch order read the same pages (with
  // the heads of a key range on one XCD instead: 53 us against 50, 4 x 16384 e4m3).
  __device__ SharePlace(const PagedAttnArgs& a, int rows_of_block) {
    const int rows = a.heads_q / a.heads_kv * a.seqlen_q;
    nrb = (rows + rows_of_block - 1) / rows_of_block;
    rb_rows = min(rows_of_block, rows);
    const int groups = a.heads_kv >> a.head_shift;
    hg = blockIdx.x % groups;
    rb = blockIdx.x / groups % nrb;
    share = blockIdx.x / (groups * nrb);
  }
};

// After a share wrote its partial of sequence b (chunks [begin, begin + all)
// of the line): the last of the sequence's shares to arrive merges them.
// Every store is acknowledged (vmcnt 0) before the workgroup's ticket; no
// workgroup waits for another.
template <int D, int NT>
__device__ inline void arrive(const PagedAttnArgs& a, const SharePlace& w, const Shares& cut, int b, int begin, int all,
                              int* flag, int tid) {
  wait_vm_all();
  __syncthreads();
  const int j0 = cut.owner(begin), j1 = cut.owner(begin + all - 1);
  if (tid == 0) {
    uint32_t* const t = a.tickets + ((int64_t)b * (a.heads_kv >> a.head_shift) + w.hg) * w.nrb + w.rb;
    const bool last = __hip_atomic_fetch_add(t, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(j1 - j0);
    if (last) __hip_atomic_store(t, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = last;
  }
  __syncthreads();
  if (*flag) merge_partials<D, true>(a, b, w.hg, w.rb, w.nrb, w.rb_rows, j0, j1, tid, NT);
}

// A query row of bfloat16 in a lane's s16x8 pieces -> fp16, scaled by a power
// of two to a largest value in [2^14, 2^15).  Returns the factor that takes
// the logits back.  (A row with an infinity or NaN has no finite result.)
template <int N>
__device__ inline float bf16_row_to_f16(s16x8 (&q)[N], float top) {
  const int ex = max((int)(__float_as_uint(top) >> 23), 15);
  const float down = __uint_as_float((uint32_t)max(268 - ex, 1) << 23);  // 2^(14 - (ex - 127))
#pragma unroll
  for (int s = 0; s < N; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) q[s][e] = (short)Elem<f16_t>::from_f(Elem<bf16_t>::to_f((uint16_t)q[s][e]) * down);
  return __uint_as_float((uint32_t)(ex - 14) << 23);
}
template <int N>
__device__ inline float bf16_row_top(const s16x8 (&q)[N]) {
  float top = 0.f;
#pragma unroll
  for (int s = 0; s < N; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(Elem<bf16_t>::to_f((uint16_t)q[s][e])));
  return top;
}

template <typename Tag, int KV, int D, int PAGES>
__global__ __launch_bounds__((AttnCfg<Tag, KV, D, PAGES>::NT)) void paged_attn_kernel(PagedAttnArgs a) {
  using C = AttnCfg<Tag, KV, D, PAGES>;
  using CT = typename std::conditional<C::KV8, f16_t, Tag>::type;  // type of the products
  constexpr bool ANY = PAGES == kAnyPages;
  constexpr int NH = PAGES == kTwoPages ? 2 : 1;  // pages a chunk is described by
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4, l16 = lane & 15;
  const int group = a.heads_q / a.heads_kv, rows = group * a.seqlen_q;
  const SharePlace w(a, C::RB);
  // The group's heads, each on `streams` waves.
  const int streams = C::NW >> a.head_shift, hw = wave & ((1 << a.head_shift) - 1), stream = wave >> a.head_shift;
  const int hk = (w.hg << a.head_shift) + hw;
  const PagedWork work{a, w.rb_rows, w.rb, 5};
  const Shares cut = work.shares<ShareRule>(lane, streams);
  if (w.share >= cut.count) return;
  const int begin = cut.begin(w.share), end = cut.begin(w.share + 1);
  int b, b_begin;
  work.find(begin, cut.pad, lane, b, b_begin);

  // This lane's piece of a chunk's first rows.
  typedef const unsigned char* bytes;
  constexpr int RPI = 64 / C::PPR;  // rows of one load
  const int prow = lane / C::PPR, pcol = lane % C::PPR;
  const bytes kbase = static_cast<bytes>(a.k) + hk * a.k_stride[2], vbase = static_cast<bytes>(a.v) + hk * a.v_stride[2];
  const bytes klane = kbase + (ANY ? 0 : (prow & 15) * a.k_stride[1]) + pcol * 16;
  const bytes vlane = vbase + (ANY ? 0 : (prow & 15) * a.v_stride[1]) + pcol * 16;
  unsigned char* const ktile = smem + wave * 2 * C::TILE;
  unsigned char* const vtile = ktile + C::TILE;
  const int mask = (1 << a.shift) - 1;
  typedef const __attribute__((address_space(4))) int32_t const_i32;
  typedef const __attribute__((address_space(4))) float const_f32;
  // Strides of the scalar paths (below 2^31).
  const uint32_t k0 = (uint32_t)a.k_stride[0], k1 = (uint32_t)a.k_stride[1];
  const uint32_t v0 = (uint32_t)a.v_stride[0], v1 = (uint32_t)a.v_stride[1];
  const uint32_t ks0 = (uint32_t)a.ks_stride[0], vs0 = (uint32_t)a.vs_stride[0], t1 = (uint32_t)a.table_stride[1];
  const float* const ks_head = a.ks ? a.ks + hk * a.ks_stride[1] : nullptr;
  const float* const vs_head = a.vs ? a.vs + hk * a.vs_stride[1] : nullptr;

  for (int at = begin; at < end;) {
    const int len = work.length(b), all = work.chunks(b);
    b_begin += cut.pad;
    at = max(at, b_begin);
    const int c0 = at - b_begin, cnt = min(end, b_begin + all) - at;
    if (cnt <= 0) break;  // (the share ends before the sequence's first chunk)
    const int blocks = (len + mask) >> a.shift;           // logical blocks of the sequence
    const int listed = a.index ? a.n_index : blocks;
    const int32_t* const index = a.index ? a.index + b * a.index_stride[0] + hk * a.index_stride[1] : nullptr;
    const int32_t* const table = a.table + b * a.table_stride[0];

    // --- what a chunk's keys are ------------------------------------------
    // Two steps ahead of its use a chunk is known by its logical blocks, one
    // step by its pages.  kAnyPages: lane l describes key l % 32.
    struct Ahead {
      int logical[NH], page[NH];
    };
    struct Meta {
      uint32_t there;      // bit k: key k of the chunk is one of the sequence's
      int key0[NH];        // position of the page's first key here, or of the lane's
      float ks[NH], vs[NH];
      int64_t koff[NH], voff[NH];
    };
    auto first_key = [&](int c, int h) { return 32 * c + (ANY ? lane & 31 : 16 * h); };
    // The logical block of the listed block that holds key n of the list.
    auto logical_of = [&](int n) {
      const int at_list = n >> a.shift;
      if (!index) return at_list;
      const int64_t i = (int64_t)min(at_list, listed - 1) * a.index_stride[2];
      int l;
      if constexpr (ANY) l = index[i];
      else l = ((const_i32*)index)[i];
      return at_list < listed ? l : -1;
    };
    auto page_of = [&](int logical) {
      const int l = min(max(logical, 0), a.max_blocks - 1);
      if constexpr (ANY) return table[l * a.table_stride[1]];
      else return ((const_i32*)table)[(uint64_t)(uint32_t)l * t1];
    };
    auto describe = [&](int c, const Ahead& x) -> Meta {
      Meta m;
      m.there = 0;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int inside = first_key(c, h) & mask;
        const bool ok = (uint32_t)x.logical[h] < (uint32_t)blocks && (uint32_t)x.page[h] < (uint32_t)a.num_blocks;
        const int page = ok ? x.page[h] : 0;
        m.key0[h] = (x.logical[h] << a.shift) + inside;
        const int here = ok ? len - m.key0[h] : 0;  // keys from this one on
        m.ks[h] = m.vs[h] = 1.f;
        if constexpr (ANY) {
          m.koff[h] = page * a.k_stride[0] + inside * a.k_stride[1];
          m.voff[h] = page * a.v_stride[0] + inside * a.v_stride[1];
          if constexpr (C::KV8) {
            if (a.ks) m.ks[h] = ks_head[page * a.ks_stride[0]];
            if (a.vs) m.vs[h] = vs_head[page * a.vs_stride[0]];
          }
          m.there = (uint32_t)__builtin_amdgcn_ballot_w64(here > 0);
        } else {
          m.koff[h] = (int64_t)((uint64_t)(uint32_t)page * k0 + (uint64_t)(uint32_t)inside * k1);
          m.voff[h] = (int64_t)((uint64_t)(uint32_t)page * v0 + (uint64_t)(uint32_t)inside * v1);
          if constexpr (C::KV8) {
            if (a.ks) m.ks[h] = ((const_f32*)ks_head)[(uint64_t)(uint32_t)page * ks0];
            if (a.vs) m.vs[h] = ((const_f32*)vs_head)[(uint64_t)(uint32_t)page * vs0];
          }
          constexpr int W = NH == 2 ? 16 : 32;
          m.there |= (here > 0 ? 0xFFFFFFFFu >> (32 - min(here, W)) : 0u) << (16 * h);
        }
        m.vs[h] = here > 0 ? m.vs[h] : 0.f;
      }
      return m;
    };
    auto far = [&](int64_t x, int from) {  // x of another lane
      const uint32_t lo = __shfl((uint32_t)x, from, 64), hi = __shfl((uint32_t)(x >> 32), from, 64);
      return (int64_t)(((uint64_t)hi << 32) | lo);
    };
    u32x4 kd[C::VN], vd[C::VN];
    auto load_rows = [&](u32x4 (&to)[C::VN], bytes from, const int64_t (&off)[NH], uint32_t stride) {
#pragma unroll
      for (int i = 0; i < C::VN; ++i) {
        bytes p;
        if constexpr (ANY) {
          p = from + far(off[0], (64 * i + lane) / C::PPR);
        } else if constexpr (RPI > 16) {  // both halves in one load
          p = from + (lane < 32 ? off[0] : NH == 2 ? off[NH - 1] : off[0] + 16 * (int64_t)stride);
        } else {
          constexpr int HALF = 16 / (RPI > 16 ? 16 : RPI);  // loads of 16 rows
          p = from + (NH == 2 ? off[i / HALF] + i % HALF * RPI * (int64_t)stride : off[0] + i * RPI * (int64_t)stride);
        }
        // (Nontemporal where a line is one head's alone: int8, D = 128, 166 ->
        // 154 us; D = 64, whose lines two waves read, 200 -> 217.)
        if constexpr (C::ONCE) to[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
        else to[i] = *reinterpret_cast<const u32x4*>(p);
      }
    };
    auto load = [&](const Meta& m) {
      load_rows(kd, klane, m.koff, k1);
      load_rows(vd, vlane, m.voff, v1);
    };
    const int mine = cnt > stream ? (cnt - stream + streams - 1) / streams : 0;
    auto chunk = [&](int k) { return min(c0 + stream + streams * k, c0 + cnt - 1); };
    Ahead first, next;  // of the chunk in flight and the one behind it
    int later[NH];      // logical blocks of the one after that
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      first.logical[h] = logical_of(first_key(chunk(0), h));
      next.logical[h] = logical_of(first_key(chunk(1), h));
      later[h] = logical_of(first_key(chunk(2), h));
    }

    // --- Q -----------------------------------------------------------------
    s16x8 q[C::NSTEP];
    const int row = w.rb * C::RB + l16;
    const bool valid = row < rows;
    const int g = valid ? row / a.seqlen_q : 0, m = valid ? row - g * a.seqlen_q : 0;
    const int klim = a.causal ? len - a.seqlen_q + m : INT_MAX;
    const uint16_t* const src = reinterpret_cast<const uint16_t*>(a.q) + b * a.q_stride[0] +
                                (hk * group + g) * a.q_stride[1] + m * a.q_stride[2];
#pragma unroll
    for (int s = 0; s < C::NSTEP; ++s) {
      // With paired K loads, lane group g4 covers 16 dims of a pair of steps.
      const int d = C::PAIR ? 64 * (s / 2) + 16 * g4 + 8 * (s % 2) : 32 * s + 8 * g4;
      q[s] = valid ? *reinterpret_cast<const s16x8*>(src + d) : zero_op<f16_t>();
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      first.page[h] = page_of(first.logical[h]);
      next.page[h] = page_of(next.logical[h]);
    }
    Meta ahead = describe(chunk(0), first);
    load(ahead);
    float qscale = a.scale_log2;
    if (C::KV8 && a.bf16) {
      float top = bf16_row_top(q);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      qscale *= bf16_row_to_f16(q, top);
    }
    float zero = 0.f;  // first value of Q K^T's sums
    if constexpr (KV == FA_KV_INT8) {
      const short c = (short)Elem<f16_t>::from_f(-kInt8Offset);
      const s16x8 off = {c, c, c, c, c, c, c, c};
      f32x4a x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < C::NSTEP; ++s) x = mma16x16<f16_t>(off, q[s], x);
      zero = x[0];
    }

    // --- the stream ----------------------------------------------------------
    float m_i = kFloor, l_i = 0.f;
    f32x4a acc[C::NDB];
#pragma unroll
    for (int i = 0; i < C::NDB; ++i) acc[i] = f32x4a{0.f, 0.f, 0.f, 0.f};
    uint32_t vref = 0x00800000u;  // bits of a power of two
    // Elements that are not finite: (x & ABS) + UP has the top bit set.
    constexpr uint32_t ABS = C::KV8 ? 0x7F7F7F7Fu : 0x7FFF7FFFu;
    constexpr uint32_t UP = C::KV8 ? 0x01010101u : std::is_same<CT, bf16_t>::value ? 0x00800080u : 0x04000400u;
    uint32_t odd = 0;  // such a value was left out
    // Some rows see keys of the chunk that others do not.
    auto is_mixed = [&](const Meta& m) {
      bool x = a.causal && a.seqlen_q > 1;
      if constexpr (!ANY) x = x && max(m.key0[0] + (NH == 1 ? 31 : 15), m.key0[NH - 1] + (NH == 1 ? 31 : 15)) > len - a.seqlen_q;
      return x;
    };

#pragma unroll 1
    for (int k = 0; k < mine; ++k) {
      const Meta m = ahead;
      const bool whole = m.there == 0xFFFFFFFFu;
      const bool mixed = is_mixed(m);
      // Rows that are no keys as zeros (0 * NaN would be NaN).
      if (!whole) {
#pragma unroll
        for (int i = 0; i < C::VN; ++i)
          if (!((m.there >> ((64 * i + lane) / C::PPR)) & 1u)) vd[i] = u32x4{0, 0, 0, 0};
      }
      // Values that are not finite must not reach the rows that do not see
      // their keys either: they are left out here, and added behind the loop.
      if (KV != FA_KV_INT8 && mixed) {
#pragma unroll
        for (int i = 0; i < C::VN; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t bad = ((vd[i][e] & ABS) + UP) & ~ABS;  // top bit of each such element
            vd[i][e] &= ~((bad >> (C::KV8 ? 7 : 15)) * (C::KV8 ? 0xFFu : 0xFFFFu));
            odd |= bad;
          }
      }
#pragma unroll
      for (int i = 0; i < C::VN; ++i) {
        const int row = (64 * i + lane) / C::PPR;
        *reinterpret_cast<u32x4*>(ktile + piece_off<C::PPR>(row, pcol)) = kd[i];
        if constexpr (C::KV8) *reinterpret_cast<u32x4*>(vtile + piece_off<C::PPR>(row, pcol)) = vd[i];
        else *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(vtile) + swz_off<D>(row, 8 * pcol)) = vd[i];
      }
      if (k + 1 < mine) {
        ahead = describe(chunk(k + 1), next);
        load(ahead);
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          next.logical[h] = later[h];
          next.page[h] = page_of(later[h]);
          later[h] = logical_of(first_key(chunk(k + 3), h));
        }
      }
      f32x4a s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = 16 * h + l16;
        s[h] = f32x4a{zero, zero, zero, zero};
        if constexpr (C::PAIR) {
#pragma unroll
          for (int t = 0; t < C::NSTEP; t += 2) {
            const u32x4 y = *reinterpret_cast<const u32x4*>(ktile + piece_off<C::PPR>(row, 2 * t + g4));
            const s16x8 lo = codes_to_f16<KV, true>(u32x2{y[0], y[1]}), hi = codes_to_f16<KV, true>(u32x2{y[2], y[3]});
            s[h] = mma16x16<CT>(lo, q[t], s[h]);
            s[h] = mma16x16<CT>(hi, q[t + 1], s[h]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < C::NSTEP; ++t) {
            s16x8 x;
            if constexpr (C::KV8)
              x = codes_to_f16<KV, true>(*reinterpret_cast<const u32x2*>(ktile + piece_off<C::PPR>(row, g4 / 2) + g4 % 2 * 8));
            else
              x = *reinterpret_cast<const s16x8*>(ktile + piece_off<C::PPR>(row, 4 * t + g4));
            s[h] = mma16x16<CT>(x, q[t], s[h]);
          }
        }
      }
      // Scales and positions: uniform over a page's keys, or each key's own.
      auto of_key = [&](const auto (&x)[NH], int h, int i) {
        if constexpr (ANY) return __shfl(x[0], 16 * h + 4 * g4 + i, 64);
        else return x[NH == 2 ? h : 0];
      };
      constexpr int NI = ANY ? 4 : 1;
      float ks[2][NI], wv[2][NI];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          ks[h][i] = of_key(m.ks, h, i);
          wv[h][i] = of_key(m.vs, h, i);
        }
      uint32_t scale_top = 0;
      if constexpr (C::KV8) {
        scale_top = __float_as_uint(m.vs[0]) & 0x7FFFFFFFu;
        if constexpr (ANY) {
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) scale_top = max(scale_top, (uint32_t)__shfl_xor((int)scale_top, o, 64));
        } else {
          scale_top = max(scale_top, __float_as_uint(m.vs[NH - 1]) & 0x7FFFFFFFu);
        }
        scale_top = __builtin_amdgcn_readfirstlane(scale_top);
        if (scale_top > vref) {
          const uint32_t grown = min((scale_top + 0x7FFFFFu) & 0x7F800000u, 0x7E800000u);
          const float f = __uint_as_float((uint32_t)max((int)(0x3F800000u + vref - grown), 0));
          vref = grown;
#pragma unroll
          for (int i = 0; i < C::NDB; ++i) acc[i] *= f;
        }
        const float inv = __uint_as_float(0x7F000000u - vref);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < NI; ++i) wv[h][i] *= inv;
      }
      float back[2][NI];  // takes a rounded weight back to p, where the scale kept its bits
      bool kept[2][NI];
      if constexpr (C::KV8) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            back[h][i] = __builtin_amdgcn_rcpf(wv[h][i]);
            kept[h][i] = fabsf(wv[h][i]) >= 0.03125f && fabsf(wv[h][i]) <= 1.f;
          }
      }
      const bool masked = ANY || !whole || mixed;
      s16x8 p;
      float f[2][NI];  // factor of the logits
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < NI; ++i) f[h][i] = qscale * ks[h][i];
      uint32_t seen = 0xFFu;  // this lane's keys that its row sees
      if (masked) {
        seen = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pos = ANY ? of_key(m.key0, h, i) : m.key0[NH == 2 ? h : 0] + (NH == 2 ? 0 : 16 * h) + 4 * g4 + i;
            const bool yes = ((m.there >> (16 * h + 4 * g4 + i)) & 1u) && pos <= klim;
            seen |= yes ? 1u << (4 * h + i) : 0u;
          }
      }
      f32x4a x[2];
      float top = kNegInf;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[h][i] = __builtin_fmaf(s[h][i], f[h][ANY ? i : 0], -m_i);
      auto hide = [&]() {
        if (masked) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i / 4][i % 4] = (seen >> i) & 1u ? x[i / 4][i % 4] : kNegInf;
        }
      };
      hide();
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i / 4][i % 4]);
      if (__builtin_amdgcn_ballot_w64(top > 8.f)) {
        float high = m_i;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            high = fmaxf(high, (seen >> (4 * h + i)) & 1u ? s[h][i] * f[h][ANY ? i : 0] : kNegInf);
        high = fmaxf(high, __shfl_xor(high, 16, 64));
        high = fmaxf(high, __shfl_xor(high, 32, 64));
        const float down = __builtin_amdgcn_exp2f(m_i - high);
        m_i = high;
        l_i *= down;
#pragma unroll
        for (int i = 0; i < C::NDB; ++i) acc[i] *= down;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[h][i] = __builtin_fmaf(s[h][i], f[h][ANY ? i : 0], -high);
        hide();
      }
      float e[8], y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(x[i / 4][i % 4]);
        y[i] = C::KV8 ? e[i] * wv[i / 4][ANY ? i % 4 : 0] : e[i];
      }
      if (C::KV8 && __builtin_expect(scale_top >= 0x7F800000u, 0)) {  // (0 * a scale that is not finite)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i / 4][i % 4] == kNegInf ? 0.f : y[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = (short)Elem<CT>::from_f(y[i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float z = Elem<CT>::to_f((uint16_t)p[i]);
        if constexpr (!C::KV8) l_i += z;
        else l_i += kept[i / 4][ANY ? i % 4 : 0] ? z * back[i / 4][ANY ? i % 4 : 0] : e[i];
      }
      // V^T: group g4's slots are the keys 4 g4 + 0 .. 3 and 16 + 4 g4 + 0 .. 3, as
      // in the scores.
#pragma unroll
      for (int i = 0; i < C::NDB; ++i) {
        s16x8 v;
        if constexpr (C::KV8) {
          // Lanes 2 j and 2 j + 1 of a group of 16 name the two halves of slot j's
          // row; lane l gets column l of the eight.
          typedef int i32x2a __attribute__((ext_vector_type(2)));
          typedef __attribute__((address_space(3))) i32x2a lds_i2;
          const int row = (l16 >> 3) * 16 + 4 * g4 + (l16 >> 1 & 3);
          unsigned char* const t = vtile + piece_off<C::PPR>(row, i) + 8 * (l16 & 1);
          v = codes_to_f16<KV, false>(__builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2*)t)));
        } else {
          typedef __attribute__((address_space(3))) s4a lds_s4;
          uint16_t* const t = reinterpret_cast<uint16_t*>(vtile) + swz_off<D>(4 * g4 + (l16 >> 2), 16 * i + 4 * (lane & 3));
          const s4a lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)t);
          const s4a hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(t + 16 * D));
          v = s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
        acc[i] = mma16x16<CT>(v, p, acc[i]);
      }
    }
    if (KV != FA_KV_INT8 && __builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) != 0, 0)) {
      // The values that were left out, key by key.
#pragma unroll 1
      for (int k = 0; k < mine; ++k) {
        Ahead x;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          x.logical[h] = logical_of(first_key(chunk(k), h));
          x.page[h] = page_of(x.logical[h]);
        }
        const Meta m = describe(chunk(k), x);
        if (!is_mixed(m)) continue;
#pragma unroll 1
        for (int key = 0; key < 32; ++key) {
          if (!((m.there >> key) & 1u)) continue;
          int64_t off;
          int pos;
          float vs;
          if constexpr (ANY) {
            off = far(m.voff[0], key);
            pos = __shfl(m.key0[0], key, 64);
            vs = __shfl(m.vs[0], key, 64);
          } else {
            const int h = NH == 2 && key >= 16 ? NH - 1 : 0, in = NH == 2 ? key & 15 : key;
            off = (h ? m.voff[NH - 1] : m.voff[0]) + in * (int64_t)v1;
            pos = (h ? m.key0[NH - 1] : m.key0[0]) + in;
            vs = h ? m.vs[NH - 1] : m.vs[0];
          }
#pragma unroll
          for (int i = 0; i < C::NDB; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bytes at_v = vbase + off + (16 * i + 4 * g4 + e) * C::ES;
              float f;
              if constexpr (C::KV8) f = (*at_v & 0x7F) == 0x7F ? __builtin_nanf("") : 0.f;
              else f = Elem<CT>::to_f(*reinterpret_cast<const uint16_t*>(at_v));
              if (f - f == 0.f) continue;
              if (pos <= klim) acc[i][e] += f * vs;
            }
        }
      }
    }

    // --- the waves' sums: out, or a partial ----------------------------------
    const float vscale = C::KV8 ? __uint_as_float(vref) : 1.f;
    float* const so = reinterpret_cast<float*>(smem);
    float* const sm = so + C::NW * C::RB * C::OLD;
    float* const sl = sm + C::NW * C::RB;
    __syncthreads();
    l_i += __shfl_xor(l_i, 16, 64);
    l_i += __shfl_xor(l_i, 32, 64);
    const int at_row = wave * C::RB + l16;  // (waves of a head: hw, hw + heads, ...)
    if (l16 < w.rb_rows) {
      float* const st = so + at_row * C::OLD + 4 * g4;
#pragma unroll
      for (int i = 0; i < C::NDB; ++i) *reinterpret_cast<f32x4a*>(st + 16 * i) = acc[i] * vscale;
      if (g4 == 0) {
        sm[at_row] = m_i;
        sl[at_row] = l_i;
      }
    }
    __syncthreads();
    const bool complete = cnt == all;
    const int here = min(w.rb_rows, rows - w.rb * C::RB);
    const int heads = 1 << a.head_shift;
    for (int i = tid; i < heads * here * (D / 4); i += C::NT) {
      const int d = i % (D / 4) * 4, r = i / (D / 4) % here, h = i / (D / 4 * here);
      float M = kFloor;
      for (int v = h; v < C::NW; v += heads) M = fmaxf(M, sm[v * C::RB + r]);
      float L = 0.f;
      f32x4a o = {0.f, 0.f, 0.f, 0.f};
      for (int v = h; v < C::NW; v += heads) {
        const float f = __builtin_amdgcn_exp2f(sm[v * C::RB + r] - M);
        L += sl[v * C::RB + r] * f;
        o += *reinterpret_cast<const f32x4a*>(so + (v * C::RB + r) * C::OLD + d) * f;
      }
      const int head = (w.hg << a.head_shift) + h;
      if (complete) {
        store_out(a, b, head, w.rb * C::RB + r, d, o * (L == 0.f ? 0.f : 1.f / L));
        continue;
      }
      const int64_t part = partial_row(a, 2 * w.share + (c0 == 0 ? 1 : 0), head, w.rb, w.nrb, w.rb_rows) + r;
      if (a.tickets) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), rsrc_of(a.ws_o), (int)((part * D + d) * 4), 0, kAgent);
        if (d == 0)
          __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(M), __float_as_uint(L)}, rsrc_of(a.ws_ml), (int)(part * 8), 0, kAgent);
      } else {
        *reinterpret_cast<f32x4a*>(a.ws_o + part * D + d) = o;
        if (d == 0) {
          a.ws_ml[2 * part] = M;
          a.ws_ml[2 * part + 1] = L;
        }
      }
    }
    if (!complete && a.tickets)
      arrive<D, C::NT>(a, w, cut, b, b_begin, all, reinterpret_cast<int*>(smem + C::LDS_BYTES - 16), tid);
    __syncthreads();  // the next sequence's tiles
    at += cnt;
    b_begin += all;
    ++b;
  }
}

// The merge as a launch of its own: grid (head groups * row blocks, batch, any).
// RB, UNIT and STREAMS: rows of a row block, log2 of a chunk's keys and chunks at
// a time (with one KV head; less with more) of the kernel that wrote the partials.
template <int D, int RB, int UNIT, int STREAMS, typename RULE>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs a) {
  const int lane = threadIdx.x & 63, b = blockIdx.y;
  const SharePlace w(a, RB);
  const PagedWork work{a, w.rb_rows, w.rb, UNIT};
  const Shares cut = work.shares<RULE>(lane, STREAMS >> a.head_shift);
  int begin = 0;
  for (int b0 = 0; b0 < b; b0 += 64) begin += b0 + lane < b ? work.chunks(b0 + lane) : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) begin += __shfl_xor(begin, o, 64);
  begin += cut.pad * (b + 1);
  const int j0 = cut.owner(begin), j1 = cut.owner(begin + work.chunks(b) - 1);
  if (j0 != j1)
    merge_partials<D, false>(a, b, w.hg, w.rb, w.nrb, w.rb_rows, j0, j1, blockIdx.z * 256 + threadIdx.x, gridDim.z * 256);
}

}  // namespace fa
