// fa_paged_attn.hip - launches of the paged attention over block scales and
// listed blocks (fa_paged_attn.hpp).
#include "fa_paged_attn.hpp"

namespace fa {

namespace {

int log2_floor(int n) {
  int s = 0;
  while ((2 << s) <= n) ++s;
  return s;
}

// KV heads of a workgroup, as a power of two: as many as fill 256 bytes of a
// token's row, where they divide the count and leave every head a wave.
int head_shift(const fa_paged_blocks_params& p, int waves) {
  int s = 0;
  const int row = p.head_dim * (p.kv_format == FA_KV_SAME ? 2 : 1);
  while ((row << s) < 256 && p.heads_kv % (2 << s) == 0 && (2 << s) <= waves) ++s;
  return s;
}

PageMode page_mode(const fa_paged_blocks_params& p) {
  const int es = p.kv_format == FA_KV_SAME ? 2 : 1;
  auto small = [](int64_t bytes) { return bytes >= 0 && bytes < (int64_t(1) << 31); };
  const bool plain = small(p.k_stride[0] * es) && small(p.k_stride[1] * es) && small(p.v_stride[0] * es) &&
                     small(p.v_stride[1] * es) && small(p.k_scale_stride[0]) && small(p.v_scale_stride[0]) &&
                     small(p.block_table_stride[1]);
  return !plain || p.block_size < 16 ? kAnyPages : p.block_size == 16 ? kTwoPages : kOnePage;
}

// Packed query rows of a KV head from which the kernel for many rows runs; below,
// blocks of 16 rows each read the cache again, from L2.  (int8, 32/8 heads of 128,
// 4 sequences up to 8192 keys: 32 rows 41 us against 42, 48 rows 49 against 43, 64
// rows 50 against 39; e4m3, 16 up to 2000: 24 rows 27.5 against 45, 48 rows 47.5
// against 49.5, 64 rows 50 against 35.)
constexpr int kManyRows = 64;

struct Plan {
  PageMode pages;
  bool many_rows;  // the kernel of fa_paged_rows.hip
  int nrb, rb_rows, shares, head_shift;
};

Plan plan_of(const fa_paged_blocks_params& p) {
  Plan w;
  w.pages = page_mode(p);
  const int64_t rows = (int64_t)(p.heads_q / p.heads_kv) * p.seqlen_q;
  const bool eight = p.kv_format != FA_KV_SAME;
  w.many_rows = eight && w.pages != kAnyPages && (p.head_dim == 64 || p.head_dim == 128) && rows >= kManyRows;
  const int rb = w.many_rows ? kRowsBlock : 16;
  w.nrb = (int)((rows + rb - 1) / rb);
  w.rb_rows = (int)std::min<int64_t>(rows, rb);
  w.head_shift = w.many_rows ? 0 : head_shift(p, 8);  // (rows below 256 bytes: 8 waves)
  // One workgroup of 8 waves, or two of 4, for each compute unit.
  const int64_t columns = (int64_t)(p.heads_kv >> w.head_shift) * w.nrb;
  const int64_t room = (int64_t)device_cu_count() * (w.many_rows ? 2 : 1);
  w.shares = p.shares > 0 ? p.shares : (int)std::max<int64_t>(1, (room + columns - 1) / columns);
  return w;
}

int64_t partial_rows(const fa_paged_blocks_params& p, const Plan& w) {
  return 2 * (int64_t)w.shares * p.heads_kv * w.nrb * w.rb_rows;
}

template <typename Tag, int KV, int D, int PAGES>
hipError_t run(PagedAttnArgs a, const Plan& w, hipStream_t stream) {
  using C = AttnCfg<Tag, KV, D, PAGES>;
  auto kern = paged_attn_kernel<Tag, KV, D, PAGES>;
  hipError_t e = allow_lds((const void*)kern, C::LDS_BYTES);
  if (e != hipSuccess) return e;
  const int columns = (a.heads_kv >> a.head_shift) * w.nrb;
  hipLaunchKernelGGL(kern, dim3((unsigned)(columns * w.shares)), dim3(C::NT), C::LDS_BYTES, stream, a);
  e = hipGetLastError();
  if (e != hipSuccess || a.tickets || w.shares == 1) return e;
  hipLaunchKernelGGL((paged_merge_kernel<D, C::RB, 5, C::NW, ShareRule>), dim3((unsigned)columns, (unsigned)a.batch), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

template <typename Tag, int KV, int D>
hipError_t run_dim(const PagedAttnArgs& a, const Plan& w, hipStream_t s) {
  switch (w.pages) {
    case kOnePage: return run<Tag, KV, D, kOnePage>(a, w, s);
    case kTwoPages: return run<Tag, KV, D, kTwoPages>(a, w, s);
    case kAnyPages: return run<Tag, KV, D, kAnyPages>(a, w, s);
  }
  return hipErrorInvalidValue;
}

template <typename Tag, int KV>
hipError_t run_format(const PagedAttnArgs& a, const Plan& w, int dim, hipStream_t s) {
  switch (dim) {
    case 32: return run_dim<Tag, KV, 32>(a, w, s);
    case 64: return run_dim<Tag, KV, 64>(a, w, s);
    case 128: return run_dim<Tag, KV, 128>(a, w, s);
    case 256: return run_dim<Tag, KV, 256>(a, w, s);
    case 512: return run_dim<Tag, KV, 512>(a, w, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

size_t paged_blocks_workspace_bytes(const fa_paged_blocks_params& p) {
  const Plan w = plan_of(p);
  return (size_t)partial_rows(p, w) * (p.head_dim + 2) * sizeof(float);
}

hipError_t launch_paged_blocks(const fa_paged_blocks_params& p, hipStream_t s) {
  const Plan w = plan_of(p);
  // The kernel's grid is one row of workgroups.
  if ((int64_t)p.heads_kv * w.nrb * w.shares > INT_MAX) return hipErrorInvalidValue;
  PagedAttnArgs a{};
  a.q = p.q;
  a.out = p.out;
  a.k = p.k_cache;
  a.v = p.v_cache;
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = p.q_stride[i];
    a.out_stride[i] = p.out_stride[i];
    a.k_stride[i] = p.k_stride[i] * (p.kv_format == FA_KV_SAME ? 2 : 1);
    a.v_stride[i] = p.v_stride[i] * (p.kv_format == FA_KV_SAME ? 2 : 1);
    a.index_stride[i] = p.block_index_stride[i];
  }
  a.table = p.block_table;
  a.lens = p.context_lens;
  a.lens_stride = p.context_lens_stride;
  a.ks = p.k_scale;
  a.vs = p.v_scale;
  for (int i = 0; i < 2; ++i) {
    a.table_stride[i] = p.block_table_stride[i];
    a.ks_stride[i] = p.k_scale_stride[i];
    a.vs_stride[i] = p.v_scale_stride[i];
  }
  a.index = p.block_index;
  a.n_index = p.n_index;
  a.num_blocks = p.num_blocks;
  a.max_blocks = p.max_blocks;
  a.shift = log2_floor(p.block_size);
  a.batch = p.batch;
  a.heads_q = p.heads_q;
  a.heads_kv = p.heads_kv;
  a.seqlen_q = p.seqlen_q;
  a.bf16 = p.dtype == FA_DTYPE_BF16;
  a.scale_log2 = p.softmax_scale * kLog2e;
  a.causal = p.causal;
  a.shares = w.shares;
  a.head_shift = w.head_shift;
  a.ws_o = reinterpret_cast<float*>(p.workspace);
  a.ws_ml = a.ws_o + partial_rows(p, w) * p.head_dim;
  // (The merge in the same launch addresses partials by 32-bit offsets.)
  a.tickets = partial_rows(p, w) * p.head_dim * 4 < (int64_t(1) << 31) ? p.tickets : nullptr;
  if (w.many_rows) return launch_paged_rows(a, p.kv_format, p.head_dim, w.nrb, s);
  // (8-bit caches: the kernels' products are fp16 for either query type.)
  switch (p.kv_format) {
    case FA_KV_E4M3: return run_format<f16_t, FA_KV_E4M3>(a, w, p.head_dim, s);
    case FA_KV_INT8: return run_format<f16_t, FA_KV_INT8>(a, w, p.head_dim, s);
    case FA_KV_SAME:
      return a.bf16 ? run_format<bf16_t, FA_KV_SAME>(a, w, p.head_dim, s) : run_format<f16_t, FA_KV_SAME>(a, w, p.head_dim, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace fa
