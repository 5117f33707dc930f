// fa_paged.hip - block tables and slot maps, appends to a paged cache, and the
// choice of blocks by their key bounds, for gfx950.  The attention that reads
// such a cache is in fa_paged_attn.hpp.
//
// The reference takes ready tables and a filled 16-bit cache
// (fa_rdna3/interface.py:643-728); nothing here has a counterpart there.
#include "fa_internal.hpp"
#include "fa_tiles.hpp"

namespace fa {

// ---------------------------------------------------------------------------
// Block tables and slot maps.
//
// With P = block_size and cap = max_blocks * P, sequence b owns the blocks
// [0, first_b) and needs [first_b, last_b), first_b = ceil(min(ctx, cap) / P),
// last_b = ceil(min(ctx + new, cap) / P); its new blocks are the free list's
// entries [start_b, start_b + last_b - first_b), start_b the running sum of
// what the sequences before it need.  Threads of the slot map read the entries
// below first_b only, and find the others in the free list: no thread reads an
// entry that another one writes.  What is done is bounded by the tensors' sizes
// (num_tokens slots, batch * max_blocks entries), whatever the lengths say.
//
// One launch, no communication between workgroups: each sums the lengths
// again (8 bytes a sequence, from L2 after the first) in windows of kSeqs
// sequences held in LDS, and looks its tokens' sequences up there.  Latency
// bounds it: 4.3 us for 64 sequences of one token, 8.6 for 300 of up to 2048
// (2.7 MB; one workgroup for 1024 tokens), against 8.3 us of host time a call.
// ---------------------------------------------------------------------------
namespace {
constexpr int kAllocThreads = 256;
constexpr int kSeqs = 1024;  // sequences of a window
}  // namespace

__global__ __launch_bounds__(kAllocThreads) void paged_allocate_kernel(fa_allocate_params p, int shift) {
  __shared__ int64_t tok_end[kSeqs];    // running sum of new tokens, sequence included
  __shared__ int64_t blk_start[kSeqs];  // running sum of needed blocks, sequence excluded
  __shared__ int64_t wave_tok[4], wave_blk[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t P = p.block_size, cap = (int64_t)p.max_blocks * P;
  const int64_t head = p.free_head ? max(*p.free_head, 0) : 0;
  const int64_t stride = (int64_t)gridDim.x * kAllocThreads;
  int64_t tok_base = 0, blk_base = 0;
  int64_t t = (int64_t)blockIdx.x * kAllocThreads + tid, u = t;  // this thread's next token and block
  for (int b0 = 0; b0 < p.batch; b0 += kSeqs) {
    constexpr int PER = kSeqs / kAllocThreads;
    int64_t tok[PER], blk[PER], tsum = 0, bsum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = b0 + tid * PER + i;
      int64_t ctx = 0, add = 0;
      if (b < p.batch) {
        ctx = max(p.context_lens[b * p.context_lens_stride], 0);
        add = max(p.new_lens[b * p.new_lens_stride], 0);
      }
      const int64_t first = (min(ctx, cap) + P - 1) >> shift, last = (min(ctx + add, cap) + P - 1) >> shift;
      blk[i] = bsum;
      tsum += add;
      bsum += last - first;
      tok[i] = tsum;
    }
    int64_t ti = tsum, bi = bsum;  // inclusive over the wave's lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t ty = __shfl_up(ti, o, 64), by = __shfl_up(bi, o, 64);
      if (lane >= o) { ti += ty; bi += by; }
    }
    if (lane == 63) { wave_tok[wave] = ti; wave_blk[wave] = bi; }
    __syncthreads();
    int64_t tprev = tok_base + ti - tsum, bprev = blk_base + bi - bsum, tall = 0, ball = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) { tprev += wave_tok[w]; bprev += wave_blk[w]; }
      tall += wave_tok[w];
      ball += wave_blk[w];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      tok_end[tid * PER + i] = tprev + tok[i];
      blk_start[tid * PER + i] = bprev + blk[i];
    }
    __syncthreads();
    if (blockIdx.x == 0) {
      if (b0 == 0 && tid == 0) p.cu_seqlens[0] = 0;
      for (int i = tid; i < kSeqs && b0 + i < p.batch; i += kAllocThreads) p.cu_seqlens[b0 + i + 1] = (int32_t)min(tok_end[i], (int64_t)INT32_MAX);
    }
    tok_base += tall;
    blk_base += ball;
    const int seqs = min(kSeqs, p.batch - b0);
    for (; u < blk_base; u += stride) {
      int lo = 0, hi = seqs - 1;  // the last sequence that starts at or before u: the one that needs it
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (blk_start[mid] <= u) lo = mid;
        else hi = mid - 1;
      }
      const int b = b0 + lo;
      const int64_t first = (min((int64_t)max(p.context_lens[b * p.context_lens_stride], 0), cap) + P - 1) >> shift;
      p.block_table[b * p.block_table_stride[0] + (first + u - blk_start[lo]) * p.block_table_stride[1]] =
          head + u < p.num_free ? p.free_blocks[(head + u) * p.free_blocks_stride] : -1;
    }
    for (; t < min(tok_base, (int64_t)p.num_tokens); t += stride) {
      int lo = 0, hi = seqs - 1;  // the first sequence that ends past t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (tok_end[mid] > t) hi = mid;
        else lo = mid + 1;
      }
      const int b = b0 + lo;
      const int64_t ctx = max(p.context_lens[b * p.context_lens_stride], 0);
      const int64_t add = max(p.new_lens[b * p.new_lens_stride], 0);
      const int64_t pos = ctx + (t - (tok_end[lo] - add));
      int64_t slot = -1;
      if (pos < cap) {
        const int64_t blk_at = pos >> shift, first = (min(ctx, cap) + P - 1) >> shift;
        int32_t page = -1;
        if (blk_at < first) {
          page = p.block_table[b * p.block_table_stride[0] + blk_at * p.block_table_stride[1]];
        } else {
          const int64_t at = head + blk_start[lo] + (blk_at - first);
          if (at < p.num_free) page = p.free_blocks[at * p.free_blocks_stride];
        }
        if (page >= 0) slot = (int64_t)page * P + (pos & (P - 1));
      }
      p.slots[t] = slot;
    }
    __syncthreads();  // the next window writes the arrays
  }
  for (; t < p.num_tokens; t += stride) p.slots[t] = -1;
  if (blockIdx.x == 0 && tid == 0) p.next_head[0] = (int32_t)min(head + blk_base, (int64_t)INT32_MAX);
}

static int log2_of(int n) {
  int s = 0;
  while ((1 << s) < n) ++s;
  return s;
}

hipError_t launch_allocate(const fa_allocate_params& p, hipStream_t stream) {
  const int64_t want = ((int64_t)p.num_tokens + 4 * kAllocThreads - 1) / (4 * kAllocThreads);
  const int grid = (int)std::min<int64_t>(std::max<int64_t>(want, 1), 1024);
  hipLaunchKernelGGL(paged_allocate_kernel, dim3(grid), dim3(kAllocThreads), 0, stream, p, log2_of(p.block_size));
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Append.  The tokens of one block (a segment: they lie within P consecutive
// rows, between them at most dropped ones) are one wave's work for each head
// of K and of V: lanes own 8 dims (16 bytes) of a row, D / 8 lanes a row, and
// 512 / D rows go at a time.  The wave of the segment's first row does it all;
// the P rows before tell whether a row is the first.
//
// 8-bit rows are x / s with s a power of two, so the quotient is exact and a
// value is rounded once, when it is stored; a block whose scale grows rounds
// its rows again on the coarser grid.  Scales of any value would round every
// row again whenever a slightly larger value arrived.
//
// Few rows: the chain slot -> old scale -> row -> store, 6 us for 64 tokens of
// 8 heads of 128.  Many: 16 prompts of up to 2048 tokens into int8, 88 MB, 25.6
// us, 3.4 TB/s; a wave's reads all come before its stores, since the scale is
// known last (rows held in registers; read again instead: 44 us).
// ---------------------------------------------------------------------------
namespace {
constexpr int kAppendWaves = 4;

struct AppendSide {
  const uint16_t* src;
  void* dst;
  float* scale;
  int64_t src_stride[2];  // token, head
  int64_t dst_stride[3];  // block, position, head
  int64_t scale_stride[2];
};

struct AppendArgs {
  AppendSide side[2];  // K, V
  const int64_t* slots;
  int64_t slots_stride;
  uint16_t* bounds;
  int64_t bounds_stride[3];  // block, head, low / high
  int32_t num_tokens, heads_kv, num_blocks, shift, chunk;
};

template <int FMT> struct Code;
template <> struct Code<FA_KV_E4M3> {
  static constexpr float kTop = 448.f;
  static constexpr int kTopExp = 8;
  static constexpr uint32_t kTopMant = 0x600000u;
  // Four codes of x * inv, |x * inv| <= top.
  __device__ static uint32_t pack_finite(const float* x, float inv) {
    const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
    return pack(y);
  }
  // Four codes of |x| <= top or NaN.
  __device__ static uint32_t pack(const float* x) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
  }
  __device__ static void unpack(uint32_t w, float* x) {
    x[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
    x[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
    x[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
  }
};
template <> struct Code<FA_KV_INT8> {
  static constexpr float kTop = 127.f;
  static constexpr int kTopExp = 6;
  static constexpr uint32_t kTopMant = 0x7E0000u;
  // Added to 1.5 * 2^23 a value is rounded to a whole number in the low bits.
  __device__ static uint32_t pack_finite(const float* x, float inv) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(__builtin_fmaf(x[i], inv, 12582912.f));
    const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000C0Cu);
    return lo | hi;
  }
  __device__ static uint32_t pack(const float* x) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)(x[i] == x[i] ? rintf(x[i]) : 0.f) & 0xFFu) << (8 * i);
    return w;
  }
  __device__ static void unpack(uint32_t w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  }
};

// x clamped to +-top; NaN stays NaN.
template <int FMT> __device__ inline float clamp_code(float x) {
  return x == x ? fminf(fmaxf(x, -Code<FMT>::kTop), Code<FMT>::kTop) : x;
}

// The least power of two 2^e, e >= -100, with amax <= top * 2^e.
template <int FMT> __device__ inline float scale_for(float amax) {
  using C = Code<FMT>;
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - C::kTopExp + ((bits & 0x7FFFFFu) > C::kTopMant ? 1 : 0);
  return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}
}  // namespace

template <typename Tag, int FMT, int D>
__global__ __launch_bounds__(64 * kAppendWaves) void paged_append_kernel(AppendArgs a) {
  using EL = Elem<Tag>;
  constexpr int LPR = D / 8;    // lanes of a row
  constexpr int RPI = 64 / LPR; // rows at a time
  extern __shared__ int32_t staged[];  // page, position of the chunk's tokens and those behind it
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int P = 1 << a.shift;
  // Neighbouring workgroups take the heads of the same tokens, K's, then V's.
  const int groups = (2 * a.heads_kv + kAppendWaves - 1) / kAppendWaves;
  const int64_t t0 = (int64_t)(blockIdx.x / groups) * a.chunk;
  // Token t0 - P + i at entry i: the chunk, and P rows before and behind it.
  const int span = a.chunk + 2 * P;
  int32_t* const page_of = staged;
  int32_t* const pos_of = staged + span;
  for (int i = tid; i < span; i += 64 * kAppendWaves) {
    const int64_t t = t0 - P + i;
    int32_t page = -1, pos = 0;
    if (t >= 0 && t < a.num_tokens) {
      const int64_t slot = a.slots[t * a.slots_stride];
      if (slot >= 0 && (slot >> a.shift) < a.num_blocks) {
        page = (int32_t)(slot >> a.shift);
        pos = (int32_t)(slot & (P - 1));
      }
    }
    page_of[i] = page;
    pos_of[i] = pos;
  }
  __syncthreads();
  const int item = blockIdx.x % groups * kAppendWaves + wave;
  if (item >= 2 * a.heads_kv) return;
  const bool is_key = item < a.heads_kv;
  const int head = is_key ? item : item - a.heads_kv;
  const AppendSide& s = a.side[is_key ? 0 : 1];
  const int c = lane % LPR, sub = lane / LPR;
  // Page and entry of the last row that is not dropped, within the P rows before.
  int prev = -1, prev_at = -1;
  for (int i0 = 0; i0 < P; i0 += 64) {
    const int at = i0 + lane < P ? page_of[i0 + lane] : -1;
    const uint64_t kept = __builtin_amdgcn_ballot_w64(at >= 0);
    if (kept) {
      prev_at = i0 + 63 - __builtin_clzll(kept);
      prev = __builtin_amdgcn_readlane(at, 63 - __builtin_clzll(kept));
    }
  }
  // The first rows of segments among the chunk's (at most 64): those that no
  // row of the same page precedes within P rows, dropped ones left out.
  uint64_t leaders;
  {
    const int at = lane < a.chunk ? page_of[P + lane] : -1;
    const uint64_t kept = __builtin_amdgcn_ballot_w64(at >= 0), under = kept & ((1ull << lane) - 1);
    const int from = under ? 63 - __builtin_clzll(under) : 0;
    const int there = __shfl(at, from, 64);  // (every lane takes part)
    const int page_before = under ? there : prev, entry_before = under ? P + from : prev_at;
    leaders = __builtin_amdgcn_ballot_w64(at >= 0 && !(at == page_before && P + lane - entry_before < P));
  }
  for (; leaders; leaders &= leaders - 1) {
    const int i = P + (int)__builtin_ctzll(leaders);
    const int page = __builtin_amdgcn_readfirstlane(page_of[i]);
    // The segment: rows i .. i + n - 1 but for dropped ones (the last is not),
    // and its lowest position.
    int n = 1, lowest = P;
    for (int j0 = 0; j0 < P; j0 += 64) {
      const int j = j0 + lane;
      const int at = j < P ? page_of[i + j] : -1;
      const uint64_t other = __builtin_amdgcn_ballot_w64(at >= 0 && at != page);
      const uint64_t before = other ? (1ull << __builtin_ctzll(other)) - 1 : ~0ull;  // lanes of the segment
      const uint64_t own = __builtin_amdgcn_ballot_w64(at == page) & before;
      if (own) n = j0 + 64 - __builtin_clzll(own);
      if ((own >> lane) & 1u) lowest = min(lowest, pos_of[i + j]);
      if (other) break;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) lowest = min(lowest, __shfl_xor(lowest, o, 64));
    lowest = __builtin_amdgcn_readfirstlane(lowest);
    const uint16_t* const src = s.src + (t0 - P + i) * s.src_stride[0] + head * s.src_stride[1] + 8 * c;
    const bool with_bounds = a.bounds && is_key;
    // Rows r0 + sub, r0 + sub + RPI, ...: N loads in flight, `ok` the rows that are there.
    auto load = [&](auto count, int r0, s16x8 (&x)[decltype(count)::value]) -> uint32_t {
      constexpr int N = decltype(count)::value;
      uint32_t ok = 0;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int r = r0 + u * RPI + sub;
        ok |= (r < n && page_of[i + min(r, n - 1)] == page) ? 1u << u : 0u;
        x[u] = *reinterpret_cast<const s16x8*>(src + min(r, n - 1) * s.src_stride[0]);
      }
      return ok;
    };
    // |x| of 16-bit values order as whole numbers do: two maxima at a time.
    // Infinities and NaN, which have no part in the scale, are the largest: a
    // segment that has some is looked at again without them.
    constexpr uint32_t kExp = std::is_same<Tag, bf16_t>::value ? 0x7F80u : 0x7C00u;
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 top = {0, 0};
    float amax = 0.f, low[8], high[8];
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) { low[e] = -kNegInf; high[e] = kNegInf; }
    auto look = [&](const s16x8& x, bool ok) {
      if (!ok) return;
      if constexpr (FMT != FA_KV_SAME) {
        const u32x4 y = __builtin_bit_cast(u32x4, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, y[e] & 0x7FFF7FFFu));
      }
      if (with_bounds) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = EL::to_f((uint16_t)x[e]);
          low[e] = fminf(low[e], f);  // (a NaN operand leaves the other)
          high[e] = fmaxf(high[e], f);
        }
      }
    };
    auto look_again = [&](const s16x8& x, bool ok) {
      if (!ok) return;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = fabsf(EL::to_f((uint16_t)x[e]));
        amax = fmaxf(amax, f < __builtin_inff() ? f : 0.f);
      }
    };
    // After the first look: the largest value, and whether all are finite.
    auto all_finite = [&]() -> bool {
      if constexpr (FMT == FA_KV_SAME) return true;
      const uint16_t t = top[0] > top[1] ? top[0] : top[1];
      finite = __builtin_amdgcn_ballot_w64(t >= kExp) == 0;
      if (finite) amax = EL::to_f(t);
      return finite;
    };
    float before = 0.f, after = 1.f;
    auto settle = [&]() {  // scale, rows of before, bounds
      if constexpr (FMT != FA_KV_SAME) {
        using C = Code<FMT>;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
        after = fmaxf(before, scale_for<FMT>(amax));
        if (lowest > 0 && after > before) {
          uint8_t* const dst = reinterpret_cast<uint8_t*>(s.dst) + page * s.dst_stride[0] + head * s.dst_stride[2] + 8 * c;
          const float ratio = before / after;
          for (int r = sub; r < lowest; r += RPI) {
            u32x2* const at = reinterpret_cast<u32x2*>(dst + r * s.dst_stride[1]);
            const u32x2 w = *at;
            u32x2 z;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x[4];
              C::unpack(w[h], x);
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] *= ratio;
              z[h] = C::pack(x);
            }
            *at = z;
          }
        }
        if (lane == 0) s.scale[page * s.scale_stride[0] + head * s.scale_stride[1]] = after;
      }
      if (with_bounds) {
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            low[e] = fminf(low[e], __shfl_xor(low[e], o, 64));
            high[e] = fmaxf(high[e], __shfl_xor(high[e], o, 64));
          }
        if (sub == 0) {
          uint16_t* const bl = a.bounds + page * a.bounds_stride[0] + head * a.bounds_stride[1] + 8 * c;
          s16x8 x, y;
#pragma unroll
          for (int e = 0; e < 8; ++e) { x[e] = (short)EL::from_f(low[e]); y[e] = (short)EL::from_f(high[e]); }
          *reinterpret_cast<s16x8*>(bl) = x;
          *reinterpret_cast<s16x8*>(bl + a.bounds_stride[2]) = y;
        }
      }
    };
    auto store = [&](const s16x8& x, int r) {
      const int64_t at = page * s.dst_stride[0] + head * s.dst_stride[2] + pos_of[i + r] * s.dst_stride[1] + 8 * c;
      if constexpr (FMT == FA_KV_SAME) {
        *reinterpret_cast<s16x8*>(reinterpret_cast<uint16_t*>(s.dst) + at) = x;
      } else {
        const float inv = 1.f / after;
        u32x2 z;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = EL::to_f((uint16_t)x[4 * h + e]);
          if (finite) {
            z[h] = Code<FMT>::pack_finite(f, inv);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = clamp_code<FMT>(f[e] * inv);
            z[h] = Code<FMT>::pack(f);
          }
        }
        *reinterpret_cast<u32x2*>(reinterpret_cast<uint8_t*>(s.dst) + at) = z;
      }
    };
    // What was there before, asked for along with the rows.
    if (lowest > 0) {
      if constexpr (FMT != FA_KV_SAME) before = s.scale[page * s.scale_stride[0] + head * s.scale_stride[1]];
      if (with_bounds && sub == 0) {
        const uint16_t* const bl = a.bounds + page * a.bounds_stride[0] + head * a.bounds_stride[1] + 8 * c;
        const s16x8 x = *reinterpret_cast<const s16x8*>(bl), y = *reinterpret_cast<const s16x8*>(bl + a.bounds_stride[2]);
#pragma unroll
        for (int e = 0; e < 8; ++e) { low[e] = EL::to_f((uint16_t)x[e]); high[e] = EL::to_f((uint16_t)y[e]); }
      }
    }
    // Up to N loads of rows stay in registers between the two looks at them.
    auto whole = [&](auto count) {
      constexpr int N = decltype(count)::value;
      s16x8 x[N];
      const uint32_t ok = load(count, 0, x);
#pragma unroll
      for (int u = 0; u < N; ++u) look(x[u], (ok >> u) & 1u);
      if (!all_finite()) {
#pragma unroll
        for (int u = 0; u < N; ++u) look_again(x[u], (ok >> u) & 1u);
      }
      settle();
      // (The rows as new values: the compiler would otherwise keep their 32-bit
      // forms from one look to the other, 230 registers in all.)
#pragma unroll
      for (int u = 0; u < N; ++u) asm("" : "+v"(x[u]));
#pragma unroll
      for (int u = 0; u < N; ++u)
        if ((ok >> u) & 1u) store(x[u], u * RPI + sub);
    };
    if (n <= RPI) {
      whole(std::integral_constant<int, 1>{});
    } else if (n <= 16 * RPI) {
      whole(std::integral_constant<int, 16>{});
    } else {
      using Eight = std::integral_constant<int, 8>;
      s16x8 x[8];
      for (int r0 = 0; r0 < n; r0 += 8 * RPI) {
        const uint32_t ok = load(Eight{}, r0, x);
#pragma unroll
        for (int u = 0; u < 8; ++u) look(x[u], (ok >> u) & 1u);
      }
      if (!all_finite()) {
        for (int r0 = 0; r0 < n; r0 += 8 * RPI) {
          const uint32_t ok = load(Eight{}, r0, x);
#pragma unroll
          for (int u = 0; u < 8; ++u) look_again(x[u], (ok >> u) & 1u);
        }
      }
      settle();
      for (int r0 = 0; r0 < n; r0 += 8 * RPI) {
        const uint32_t ok = load(Eight{}, r0, x);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if ((ok >> u) & 1u) store(x[u], r0 + u * RPI + sub);
      }
    }
  }
}

template <typename Tag, int FMT, int D>
static hipError_t run_append(const AppendArgs& a, hipStream_t stream) {
  const int64_t groups = (2 * a.heads_kv + kAppendWaves - 1) / kAppendWaves;
  const int64_t grid = groups * (((int64_t)a.num_tokens + a.chunk - 1) / a.chunk);
  if (grid > INT_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL((paged_append_kernel<Tag, FMT, D>), dim3((unsigned)grid), dim3(64 * kAppendWaves),
                     2 * (a.chunk + (2 << a.shift)) * sizeof(int32_t), stream, a);
  return hipGetLastError();
}

template <typename Tag, int FMT>
static hipError_t append_by_dim(const AppendArgs& a, int dim, hipStream_t stream) {
  switch (dim) {
    case 16: return FMT == FA_KV_SAME ? run_append<Tag, FA_KV_SAME, 16>(a, stream) : hipErrorInvalidValue;
    case 32: return run_append<Tag, FMT, 32>(a, stream);
    case 64: return run_append<Tag, FMT, 64>(a, stream);
    case 128: return run_append<Tag, FMT, 128>(a, stream);
    case 256: return run_append<Tag, FMT, 256>(a, stream);
    case 512: return run_append<Tag, FMT, 512>(a, stream);
  }
  return hipErrorInvalidValue;
}

template <typename Tag>
static hipError_t append_by_format(const AppendArgs& a, int format, int dim, hipStream_t stream) {
  switch (format) {
    case FA_KV_SAME: return append_by_dim<Tag, FA_KV_SAME>(a, dim, stream);
    case FA_KV_E4M3: return append_by_dim<Tag, FA_KV_E4M3>(a, dim, stream);
    case FA_KV_INT8: return append_by_dim<Tag, FA_KV_INT8>(a, dim, stream);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_paged_append(const fa_paged_append_params& p, hipStream_t stream) {
  if (p.num_tokens == 0) return hipSuccess;
  AppendArgs a{};
  auto side = [&](AppendSide& s, const void* src, void* dst, float* scale, const int64_t* ss, const int64_t* ds,
                  const int64_t* cs) {
    s.src = reinterpret_cast<const uint16_t*>(src);
    s.dst = dst;
    s.scale = scale;
    for (int i = 0; i < 2; ++i) s.src_stride[i] = ss[i];
    for (int i = 0; i < 3; ++i) s.dst_stride[i] = ds[i];
    for (int i = 0; i < 2; ++i) s.scale_stride[i] = cs[i];
  };
  side(a.side[0], p.k_new, p.k_cache, p.k_scale, p.k_new_stride, p.k_cache_stride, p.k_scale_stride);
  side(a.side[1], p.v_new, p.v_cache, p.v_scale, p.v_new_stride, p.v_cache_stride, p.v_scale_stride);
  a.slots = p.slots;
  a.slots_stride = p.slots_stride;
  a.bounds = reinterpret_cast<uint16_t*>(p.key_bounds);
  for (int i = 0; i < 3; ++i) a.bounds_stride[i] = p.bounds_stride[i];
  a.num_tokens = p.num_tokens;
  a.heads_kv = p.heads_kv;
  a.num_blocks = p.num_blocks;
  a.shift = log2_of(p.block_size);
  // Tokens of a workgroup: one while the chip is not full of waves (16 a compute
  // unit), then more, up to a block's worth, since most tokens of a long prompt
  // lead no segment.  (With 64 a unit instead: 16-bit chunks of 333 tokens 12.8 us
  // against 7.9, prompts 25 against 16, 64 x 20 tokens of e4m3 10.6 against 12.2;
  // with 4: 9.6, 16, 20.6.)
  const int64_t waves = (int64_t)p.num_tokens * 2 * p.heads_kv;
  a.chunk = 1;
  while (a.chunk < p.block_size && a.chunk < 64 && waves / a.chunk > 16 * (int64_t)device_cu_count()) a.chunk *= 2;
  return p.dtype == FA_DTYPE_F16 ? append_by_format<f16_t>(a, p.kv_format, p.head_dim, stream)
                                 : append_by_format<bf16_t>(a, p.kv_format, p.head_dim, stream);
}

// ---------------------------------------------------------------------------
// Choice of blocks.  The score sum_d max(q_d, 0) hi_d + min(q_d, 0) lo_d is at
// least q.k for every key within the bounds.  Sums are in 64 bits (products of
// two 16-bit values are exact there), so that a block at the border does not
// depend on the order of a sum.
//
// paged_score_kernel: a lane owns 8 dims of a block (16 bytes of each bound)
// and 4 query rows in registers, D / 8 lanes a block; a wave asks for the
// bounds of several blocks at once.  The 4 rows' sums are folded over the lanes
// with the rows shared out, so that a step halves what is left to add.  Each
// block's score goes to the workspace as an integer of the same order.
// Vector instructions bound it: 32 x 8 x 2048 blocks of 128 dims and 4 rows,
// 147 MB, 47 us (3.1 TB/s), of which the 64-bit FMAs alone take 14 at full rate;
// the rest are the conversions to 64 bits, the folds and the ramp.
// paged_top_kernel: one workgroup per (sequence, KV head) finds the n_index-th
// largest by 12-bit digits and writes the chosen ones in index order; its digits
// come in turn, 8 us for 1024 blocks, 10 for 2048.  Up to 4096 keys stay in
// registers; more are read again from L2 for every digit.
// ---------------------------------------------------------------------------
namespace {
constexpr int kScoreThreads = 256;
constexpr int kScoreMost = 512;   // most blocks of a workgroup
constexpr int kScoreRows = 4;     // query rows at a time
constexpr uint64_t kAlways = ~0ull;
constexpr uint64_t kLowest = 0x000FFFFFFFFFFFFFull;  // order_of(-infinity)

struct SelectArgs {
  fa_select_params p;
  uint64_t* keys;  // (batch, heads_kv, max_blocks)
  int32_t shift;
  int32_t span;    // blocks of a scoring workgroup: 64 for each round of its waves' 16
};

// An integer that orders as the double does (NaN: as +infinity; -0 as 0).
__device__ inline uint64_t order_of(double x) {
  if (x != x) x = __builtin_inf();
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

// x of lane ^ X, for X below 16 within the vector unit: through LDS the steps of
// a sum wait for one another (32 x 8 x 2048 blocks of D = 128: 75 us against 67,
// and 64 with the reads sharing the steps as well).
template <int X> __device__ inline int of_lane_xor(int x) {
  if constexpr (X == 1) return __builtin_amdgcn_mov_dpp(x, 0xB1, 0xF, 0xF, true);  // quad_perm 1 0 3 2
  else if constexpr (X == 2) return __builtin_amdgcn_mov_dpp(x, 0x4E, 0xF, 0xF, true);  // quad_perm 2 3 0 1
  else if constexpr (X == 8) return __builtin_amdgcn_mov_dpp(x, 0x128, 0xF, 0xF, true);  // row_ror 8
  else if constexpr (X == 4) {
    const int up = __builtin_amdgcn_mov_dpp(x, 0x104, 0xF, 0xF, true);  // row_shl 4: of lane + 4
    return __builtin_amdgcn_update_dpp(up, x, 0x114, 0xF, 0xA, true);   // row_shr 4, odd groups of 4
  } else return __shfl_xor(x, X, 64);
}
template <int X> __device__ inline double of_lane_xor(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x);
  const uint64_t lo = (uint32_t)of_lane_xor<X>((int)b), hi = (uint32_t)of_lane_xor<X>((int)(b >> 32));
  return __longlong_as_double((long long)(hi << 32 | lo));
}

__device__ inline int blocks_of(const SelectArgs& a, int b) {
  const int64_t len = max(a.p.context_lens[b * a.p.context_lens_stride], 0);
  return (int)min((int64_t)a.p.max_blocks, (len + a.p.block_size - 1) >> a.shift);
}
}  // namespace

template <typename Tag, int D>
__global__ __launch_bounds__(kScoreThreads) void paged_score_kernel(SelectArgs a) {
  using EL = Elem<Tag>;
  constexpr int LPB = D / 8;                       // lanes of a block
  constexpr int BPW = 64 / LPB;                    // blocks a wave reads at a time
  constexpr int WAVES = kScoreThreads / 64;
  constexpr int OWN = 16;                          // blocks of a wave in a round
  constexpr int PER = OWN / BPW;                   // reads for them
  constexpr int AT_ONCE = PER < 4 ? PER : 4;       // reads in flight together, and as many behind them
  __shared__ uint64_t best[kScoreMost];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.y, b = blockIdx.z;
  const int n = blocks_of(a, b);
  const int first = blockIdx.x * a.span, here = min(a.span, n - first);
  // A choice is only made among more than n_index blocks.
  if (n <= a.p.n_index || here <= 0) return;
  const int group = a.p.heads_q / a.p.heads_kv, rows = group * a.p.seqlen_q;
  const int c = lane % LPB, sub = lane / LPB;
  const uint16_t* const bounds = reinterpret_cast<const uint16_t*>(a.p.key_bounds) + h * a.p.bounds_stride[1] + 8 * c;
  const int32_t* const table = a.p.block_table + b * a.p.block_table_stride[0];
  // Blocks of the workgroup: round j of wave w holds j * 64 + 16 w + 0 .. 15.
  const int rounds = (here + OWN * WAVES - 1) / (OWN * WAVES);
  auto pages_of = [&](int j) {  // one a lane, -1: none
    const int k = j * OWN * WAVES + wave * OWN + lane % OWN;
    int page = -1;
    if (j < rounds && k < here) page = table[(int64_t)(first + k) * a.p.block_table_stride[1]];
    return page < a.p.num_blocks ? page : -1;
  };
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += kScoreRows) {
    double pos[kScoreRows][8], neg[kScoreRows][8];
#pragma unroll
    for (int r = 0; r < kScoreRows; ++r) {
      const int row = min(r0 + r, rows - 1);  // (a row twice changes no maximum)
      const int g = row / a.p.seqlen_q, m = row - g * a.p.seqlen_q;
      const s16x8 q = *reinterpret_cast<const s16x8*>(reinterpret_cast<const uint16_t*>(a.p.q) + b * a.p.q_stride[0] +
                                                      (h * group + g) * a.p.q_stride[1] + m * a.p.q_stride[2] + 8 * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = EL::to_f((uint16_t)q[e]);
        pos[r][e] = x > 0.f ? (double)x : x == x ? 0.0 : (double)x;  // (NaN in both)
        neg[r][e] = x < 0.f ? (double)x : x == x ? 0.0 : (double)x;
      }
    }
    int pages = pages_of(0), pages_next = pages_of(1);
    s16x8 lo[AT_ONCE], hi[AT_ONCE];
    int page[AT_ONCE];
    auto ask = [&](int from, int i0) {
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        page[u] = __shfl(from, (i0 + u) * BPW + sub, 64);
        const uint16_t* const p = bounds + max(page[u], 0) * a.p.bounds_stride[0];
        lo[u] = *reinterpret_cast<const s16x8*>(p);
        hi[u] = *reinterpret_cast<const s16x8*>(p + a.p.bounds_stride[2]);
      }
    };
    ask(pages, 0);
#pragma unroll 1
    for (int j = 0; j < rounds; ++j) {
#pragma unroll 1
      for (int i0 = 0; i0 < PER; i0 += AT_ONCE) {
        s16x8 l_now[AT_ONCE], h_now[AT_ONCE];
        int p_now[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) { l_now[u] = lo[u]; h_now[u] = hi[u]; p_now[u] = page[u]; }
        const bool turn = i0 + AT_ONCE >= PER;
        if (turn) {
          pages = pages_next;
          pages_next = pages_of(j + 2);
        }
        ask(pages, turn ? 0 : i0 + AT_ONCE);
        // A lane's share of the sums, then the sums over the block's lanes, halved
        // at each step by what a lane keeps: by bit 0 rows {0, 1} or {2, 3}, by bit
        // 1 one of the two, by bits 2 and 3 one of the reads.
        double v[AT_ONCE];
        const bool odd = lane & 1, two = lane & 2, four = lane & 4, eight = lane & 8;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
          double sum[kScoreRows] = {};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const double l = EL::to_f((uint16_t)l_now[u][e]), g = EL::to_f((uint16_t)h_now[u][e]);
#pragma unroll
            for (int r = 0; r < kScoreRows; ++r) {
              sum[r] = __builtin_fma(pos[r][e], g, sum[r]);
              sum[r] = __builtin_fma(neg[r][e], l, sum[r]);
            }
          }
          double x[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) x[i] = (odd ? sum[i + 2] : sum[i]) + of_lane_xor<1>(odd ? sum[i] : sum[i + 2]);
          v[u] = (two ? x[1] : x[0]) + of_lane_xor<2>(two ? x[0] : x[1]);
        }
        int at = 0;  // the read whose sum this lane keeps
        if constexpr (AT_ONCE > 1) {
          constexpr int HALF = AT_ONCE / 2;
#pragma unroll
          for (int i = 0; i < HALF; ++i) v[i] = (four ? v[i + HALF] : v[i]) + of_lane_xor<4>(four ? v[i] : v[i + HALF]);
          at = four ? HALF : 0;
        }
        if constexpr (AT_ONCE > 2) {
          v[0] = (eight ? v[1] : v[0]) + of_lane_xor<8>(eight ? v[0] : v[1]);
          at += eight ? 1 : 0;
        }
        if constexpr (LPB > 16) v[0] += of_lane_xor<16>(v[0]);
        if constexpr (LPB > 32) v[0] += of_lane_xor<32>(v[0]);
        static_assert(AT_ONCE == (LPB == 4 ? 1 : LPB == 8 ? 2 : 4), "the sums end in one value a lane");
        double most = v[0] == v[0] ? v[0] : __builtin_inf();
        most = fmax(most, of_lane_xor<1>(most));
        most = fmax(most, of_lane_xor<2>(most));
        int at_page = p_now[0];
#pragma unroll
        for (int u = 1; u < AT_ONCE; ++u) at_page = at == u ? p_now[u] : at_page;
        if ((c & ~(4 * (AT_ONCE - 1))) == 0) {
          const int k = j * OWN * WAVES + wave * OWN + (i0 + at) * BPW + sub;  // block, within the workgroup's
          const uint64_t key = at_page >= 0 ? order_of(most) : kLowest;
          best[k] = r0 == 0 ? key : max(best[k], key);
        }
      }
    }
  }
  __syncthreads();
  for (int k = tid; k < here; k += kScoreThreads) {
    const int blk = first + k;
    const bool always = blk < a.p.keep_first || blk >= n - a.p.keep_last;
    a.keys[((int64_t)b * a.p.heads_kv + h) * a.p.max_blocks + blk] = always ? kAlways : best[k];
  }
}

namespace {
constexpr int kTopThreads = 1024, kTopWaves = kTopThreads / 64;
constexpr int kDigit = 12, kBins = 1 << kDigit;
}  // namespace

// PER: keys a thread holds in registers (index j * kTopThreads + thread), or 0:
// the keys are read again for every digit.
template <int PER>
__global__ __launch_bounds__(kTopThreads) void paged_top_kernel(SelectArgs a) {
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t wave_sum[kTopWaves];
  __shared__ int32_t found[2];
  constexpr int TILES = PER ? PER : 1;
  __shared__ int32_t taken[TILES * kTopWaves], equal[TILES * kTopWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x, b = blockIdx.y;
  const int n = blocks_of(a, b), want = a.p.n_index;
  int32_t* const out = a.p.index + ((int64_t)b * a.p.heads_kv + h) * want;
  if (n <= want) {
    for (int i = tid; i < want; i += kTopThreads) out[i] = i < n ? i : -1;
    return;
  }
  const uint64_t* const keys = a.keys + ((int64_t)b * a.p.heads_kv + h) * a.p.max_blocks;
  uint64_t mine[TILES];
  if constexpr (PER) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = j * kTopThreads + tid;
      mine[j] = keys[min(i, n - 1)];
    }
  }
  // The want-th largest key, digit by digit: `prefix` holds the digits found,
  // `left` how many of the keys that share them are still to be taken.
  uint64_t prefix = 0;
  int left = want;
  for (int top = 64; top > 0; top -= kDigit) {
    const int low = max(top - kDigit, 0), width = top - low;
    constexpr int BPT = kBins / kTopThreads;
    for (int i = tid; i < kBins; i += kTopThreads) bins[i] = 0;
    __syncthreads();
    auto count = [&](uint64_t k, bool there) {
      const bool in = there && (top == 64 || (k >> top) == (prefix >> top));
      const uint32_t bin = (uint32_t)(k >> low) & ((1u << width) - 1);
      // Scores share their leading digits: one atomic for all lanes of a bin,
      // for the first two bins.
      uint64_t rest = __builtin_amdgcn_ballot_w64(in);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!rest) return;
        const int lead = __builtin_ctzll(rest);
        const uint64_t same = __builtin_amdgcn_ballot_w64(bin == (uint32_t)__builtin_amdgcn_readlane((int)bin, lead)) & rest;
        if (lane == lead) atomicAdd(&bins[bin], (uint32_t)__builtin_popcountll(same));
        rest &= ~same;
      }
      if ((rest >> lane) & 1u) atomicAdd(&bins[bin], 1u);
    };
    if constexpr (PER) {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (j * kTopThreads < n) count(mine[j], j * kTopThreads + tid < n);
    } else {
      for (int i0 = 0; i0 < n; i0 += kTopThreads) count(keys[min(i0 + tid, n - 1)], i0 + tid < n);
    }
    __syncthreads();
    // Thread t sums the bins [t * BPT, (t + 1) * BPT) from the highest thread down.
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < BPT; ++i) sum += bins[tid * BPT + i];
    uint32_t above = sum;  // inclusive, over the lanes from this one up
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_down(above, o, 64);
      if (lane + o < 64) above += y;
    }
    if (lane == 0) wave_sum[wave] = above;
    __syncthreads();
    above -= sum;
    for (int w = wave + 1; w < kTopWaves; ++w) above += wave_sum[w];
    if ((int)above < left && (int)(above + sum) >= left) {
      int digit = BPT - 1;
      uint32_t seen = above;
      while ((int)(seen + bins[tid * BPT + digit]) < left) seen += bins[tid * BPT + digit--];
      found[0] = tid * BPT + digit;
      found[1] = left - (int)seen;
      taken[0] = (int)bins[tid * BPT + digit];
    }
    __syncthreads();
    prefix |= (uint64_t)found[0] << low;
    left = found[1];
    const bool done = taken[0] == left;  // every key of this digit is in
    __syncthreads();
    if (done) {
      left = INT_MAX;  // the keys from `prefix` on are the ones wanted
      break;
    }
  }
  // Keys above `prefix`, and the first `left` equal to it, in index order
  // (left INT_MAX: all that are not below it).
  const bool all = left == INT_MAX;
  auto is_eq = [&](uint64_t k) { return !all && k == prefix; };
  auto is_in = [&](uint64_t k) { return all ? k >= prefix : k > prefix; };
  const uint64_t below = (1ull << lane) - 1;
  int at = 0, eq_at = 0;
  for (int i0 = 0; i0 < n; i0 += TILES * kTopThreads) {
    // Counts of each (tile, wave), then their running sums.
    if constexpr (!PER) mine[0] = keys[min(i0 + tid, n - 1)];
#pragma unroll
    for (int j = 0; j < TILES; ++j) {
      const bool there = i0 + j * kTopThreads + tid < n;
      const uint64_t e = __builtin_amdgcn_ballot_w64(there && is_eq(mine[j])), g = __builtin_amdgcn_ballot_w64(there && is_in(mine[j]));
      if (lane == 0) {
        equal[j * kTopWaves + wave] = __builtin_popcountll(e);
        taken[j * kTopWaves + wave] = __builtin_popcountll(g);
      }
    }
    __syncthreads();
    static_assert(TILES * kTopWaves <= 64, "one lane for each (tile, wave)");
    const int my_eq = lane < TILES * kTopWaves ? equal[lane] : 0, my_in = lane < TILES * kTopWaves ? taken[lane] : 0;
    int eqs = my_eq, ins = my_in;  // inclusive sums over (tile, wave)
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(eqs, o, 64), y = __shfl_up(ins, o, 64);
      if (lane >= o) { eqs += x; ins += y; }
    }
    const int eq_all = __shfl(eqs, 63, 64), in_all = __shfl(ins, 63, 64);
    eqs -= my_eq;
    ins -= my_in;
#pragma unroll
    for (int j = 0; j < TILES; ++j) {
      const int i = i0 + j * kTopThreads + tid;
      const bool there = i < n, e = there && is_eq(mine[j]), g = there && is_in(mine[j]);
      const uint64_t eb = __builtin_amdgcn_ballot_w64(e), gb = __builtin_amdgcn_ballot_w64(g);
      const int e_before = eq_at + __shfl(eqs, j * kTopWaves + wave, 64) + __builtin_popcountll(eb & below);
      const int g_before = at + __shfl(ins, j * kTopWaves + wave, 64) + __builtin_popcountll(gb & below);
      // Equal keys before this one that are in: the first `left` of them.
      if (g || (e && e_before < left)) out[g_before + min(e_before, left)] = i;
    }
    at += in_all;
    eq_at += eq_all;
    __syncthreads();
  }
}

size_t select_workspace_bytes(int batch, int heads_kv, int max_blocks) {
  return (size_t)batch * heads_kv * max_blocks * sizeof(uint64_t);
}

template <typename Tag>
static hipError_t select_by_dim(const SelectArgs& a, hipStream_t stream) {
  const dim3 grid((a.p.max_blocks + a.span - 1) / a.span, a.p.heads_kv, a.p.batch);
  const dim3 block(kScoreThreads);
  switch (a.p.head_dim) {
    case 32: hipLaunchKernelGGL((paged_score_kernel<Tag, 32>), grid, block, 0, stream, a); break;
    case 64: hipLaunchKernelGGL((paged_score_kernel<Tag, 64>), grid, block, 0, stream, a); break;
    case 128: hipLaunchKernelGGL((paged_score_kernel<Tag, 128>), grid, block, 0, stream, a); break;
    case 256: hipLaunchKernelGGL((paged_score_kernel<Tag, 256>), grid, block, 0, stream, a); break;
    case 512: hipLaunchKernelGGL((paged_score_kernel<Tag, 512>), grid, block, 0, stream, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_select(const fa_select_params& p, hipStream_t stream) {
  SelectArgs a{};
  a.p = p;
  a.keys = reinterpret_cast<uint64_t*>(p.workspace);
  a.shift = log2_of(p.block_size);
  // A workgroup's blocks: 64 while that leaves it company on a compute unit,
  // then more, so that fewer of them convert their rows again.  (Where 8 a unit
  // would be left, 32 x 8 x 2048 blocks: 63 us, with 4 59, always 64 blocks 90;
  // 16 x 8 x 1875 of D = 64: 22 us, with 4 a unit 27.)
  a.span = 64;
  const int64_t all = (int64_t)p.batch * p.heads_kv * p.max_blocks;
  while (a.span < kScoreMost && all / a.span > 8 * (int64_t)device_cu_count()) a.span *= 2;
  if (p.max_blocks > p.n_index) {
    const hipError_t e = p.dtype == FA_DTYPE_F16 ? select_by_dim<f16_t>(a, stream) : select_by_dim<bf16_t>(a, stream);
    if (e != hipSuccess) return e;
  }
  const dim3 grid(p.heads_kv, p.batch);
  if (p.max_blocks <= kTopThreads) hipLaunchKernelGGL(paged_top_kernel<1>, grid, dim3(kTopThreads), 0, stream, a);
  else if (p.max_blocks <= 4 * kTopThreads) hipLaunchKernelGGL(paged_top_kernel<4>, grid, dim3(kTopThreads), 0, stream, a);
  else hipLaunchKernelGGL(paged_top_kernel<0>, grid, dim3(kTopThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace fa
