// The paged cache's handle, the write of new tokens into it (norm, rotary embedding, pages) and
// eviction by accumulated attention weight (include/tq4_paged.h). Attention is paged_attention.cu.
#include "paged.cuh"

namespace tq4 {

// ---- append -----------------------------------------------------------------------------------
constexpr int kAppendThreads = 256;
constexpr int kAppendMaxPairs = 128;  // head_dim <= 256

struct AppendArgs {
  PagedView cache;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  void *q_out, *k_pages, *v_pages;
  const int32_t *seq, *slot, *positions;
  int64_t tokens;
  int heads;
  const float *cos_t, *sin_t, *q_w, *k_w;
  int64_t max_pos;
  float eps;
  int pairs, axes, interleaved;
  uint8_t pair_axis[kAppendMaxPairs];
};

// A warp per row of a token: heads queries, then the keys, then the values.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_wait();
  pdl_trigger();
  const PagedView& c = a.cache;
  const int lane = threadIdx.x & 31, D = c.head_dim;
  const int rows = a.heads + 2 * c.kv_heads;
  const int64_t w = (int64_t)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int64_t t = w / rows;
  const int r = (int)(w - t * rows);
  if (t >= a.tokens) return;
  const int s = a.seq[t];
  if (s < 0) return;  // padding
  const int64_t slot = a.slot[t];
  bool ok = s < c.max_seqs && slot >= 0 && slot < c.max_slots;
  int64_t pos[4] = {0, 0, 0, 0};
  if (a.pairs > 0)
    for (int i = 0; i < a.axes; ++i) {
      pos[i] = a.positions[i * a.tokens + t];
      ok = ok && pos[i] >= 0 && pos[i] < a.max_pos;
    }
  const int page = ok ? c.table[(int64_t)s * c.max_pages + (slot >> c.page_log2)] : -1;
  if (!c.page_ok(page)) {
    if (lane == 0) report(kDevBadArgument);
    return;
  }
  const int in_page = (int)(slot & ((1 << c.page_log2) - 1));
  const T* x;
  T* y;
  const float* nw = nullptr;
  int pairs = a.pairs;
  if (r < a.heads) {
    x = static_cast<const T*>(a.q) + t * a.q_stride + (int64_t)r * D;
    y = static_cast<T*>(a.q_out) + (t * a.heads + r) * D;
    nw = a.q_w;
  } else if (r < a.heads + c.kv_heads) {
    const int h = r - a.heads;
    x = static_cast<const T*>(a.k) + t * a.k_stride + (int64_t)h * D;
    y = static_cast<T*>(a.k_pages) + c.row_offset(page, h, in_page);
    nw = a.k_w;
  } else {
    const int h = r - a.heads - c.kv_heads;
    x = static_cast<const T*>(a.v) + t * a.v_stride + (int64_t)h * D;
    y = static_cast<T*>(a.v_pages) + c.row_offset(page, h, in_page);
    pairs = 0;
  }
  float inv = 1.f;
  if (nw) {
    float ss = 0.f;
    for (int i = lane; i < D; i += 32) {
      const float v = to_f32(x[i]);
      ss = fmaf(v, v, ss);
    }
    for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    inv = 1.f / sqrtf(ss / (float)D + a.eps);
  }
  for (int i = lane; i < pairs; i += 32) {
    const int e0 = a.interleaved ? 2 * i : i, e1 = a.interleaved ? 2 * i + 1 : i + pairs;
    float x0 = to_f32(x[e0]), x1 = to_f32(x[e1]);
    if (nw) {
      x0 = x0 * inv * nw[e0];
      x1 = x1 * inv * nw[e1];
    }
    const int64_t row = pos[a.pair_axis[i]] * pairs + i;
    const float cs = a.cos_t[row], sn = a.sin_t[row];
    y[e0] = from_f32<T>(x0 * cs - x1 * sn);
    y[e1] = from_f32<T>(x1 * cs + x0 * sn);
  }
  for (int i = 2 * pairs + lane; i < D; i += 32) {
    if (nw)
      y[i] = from_f32<T>(to_f32(x[i]) * inv * nw[i]);
    else
      y[i] = x[i];
  }
}

// ---- evict ------------------------------------------------------------------------------------
constexpr int kSelectThreads = 1024;

struct EvictArgs {
  PagedView cache;
  const int32_t* lengths;
  int64_t batch;
  const float* scores;
  int64_t keep, recent;
  const int32_t* new_table;
  int32_t new_max_pages;
  int32_t *new_lengths, *kept;
  float* new_scores;
  int64_t new_score_stride;
  char *k_pages, *v_pages;
  int row_bytes;
};

// A score's place in the order: larger keys for larger scores, -0 as 0, NaN below all.
__device__ __forceinline__ uint32_t score_key(float f) {
  if (f != f) return 0;
  const uint32_t u = __float_as_uint(f + 0.f);  // -0 + 0 = 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Sum over the threads before this one, and over all of them in *total (kSelectThreads threads).
__device__ __forceinline__ int block_prefix(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, off);
      if (lane >= off) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  const int before = warp ? warp_sums[warp - 1] : 0;
  *total = warp_sums[31];
  __syncthreads();
  return before + x - v;
}

// One CTA per (sequence, KV head): the kept slots. The smallest kept score among the candidates is
// found by radix selection, eight bits of the key a pass; then one ordered pass over the slots
// takes the keys above it and the first of its equals.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ int hist[256];
  __shared__ int warp_sums[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const PagedView& c = a.cache;
  const int64_t row = blockIdx.x;
  const int64_t b = row / c.kv_heads;
  const int tid = threadIdx.x;
  const int64_t L = paged_length(c, a.lengths, b);
  const float* sc = a.scores + row * c.max_slots;
  int32_t* kept = a.kept + row * a.keep;
  float* ns = a.new_scores ? a.new_scores + row * a.new_score_stride : nullptr;
  const int64_t stay = L < a.keep ? L : a.keep;
  if (row == b * c.kv_heads && tid == 0) a.new_lengths[b] = (int32_t)stay;
  for (int64_t i = stay + tid; i < a.keep; i += kSelectThreads) kept[i] = -1;
  if (L <= a.keep) {
    for (int64_t i = tid; i < L; i += kSelectThreads) {
      kept[i] = (int32_t)i;
      if (ns) ns[i] = sc[i];
    }
    return;
  }
  const int64_t n = L - a.recent;  // candidates, more than keep - recent of them
  const int64_t most = a.keep - a.recent;
  uint32_t edge = 0xffffffffu;
  int need = 0;  // how many of the scores equal to the edge are kept
  if (most > 0) {
    uint32_t prefix = 0;
    need = (int)most;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      for (int64_t i = tid; i < n; i += kSelectThreads) {
        const uint32_t key = score_key(sc[i]);
        if (shift == 24 || ((key ^ prefix) >> (shift + 8)) == 0) atomicAdd(&hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255, left = need;
        while (d > 0 && hist[d] < left) left -= hist[d--];
        s_prefix = prefix | ((uint32_t)d << shift);
        s_need = left;
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
      __syncthreads();
    }
    edge = prefix;
  }
  int64_t placed = 0, equals = 0;
  for (int64_t base = 0; base < n && most > 0; base += kSelectThreads) {
    const int64_t i = base + tid;
    const float f = i < n ? sc[i] : 0.f;
    const uint32_t key = score_key(f);
    const bool eq = i < n && key == edge;
    int total;
    const int eq_before = block_prefix(eq, warp_sums, &total);
    const bool take = i < n && (key > edge || (eq && equals + eq_before < need));
    equals += total;
    const int at = block_prefix(take, warp_sums, &total);
    if (take) {
      kept[placed + at] = (int32_t)i;
      if (ns) ns[placed + at] = f;
    }
    placed += total;
  }
  for (int64_t i = tid; i < a.recent; i += kSelectThreads) {
    kept[most + i] = (int32_t)(n + i);
    if (ns) ns[most + i] = sc[n + i];
  }
}

// Moves the kept rows: a warp per row of K and V.
constexpr int kMoveThreads = 256;
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictArgs a) {
  pdl_wait();
  pdl_trigger();
  const PagedView& c = a.cache;
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.batch * c.kv_heads * a.keep;
  for (int64_t w = (int64_t)blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); w < rows;
       w += (int64_t)gridDim.x * (kMoveThreads / 32)) {
    const int64_t j = w % a.keep, bh = w / a.keep;
    const int64_t b = bh / c.kv_heads;
    const int h = (int)(bh - b * c.kv_heads);
    const int slot = a.kept[w];
    if (slot < 0) continue;
    const int mask = (1 << c.page_log2) - 1;
    const int from = c.table[b * c.max_pages + (slot >> c.page_log2)];
    const int to = a.new_table[b * a.new_max_pages + (j >> c.page_log2)];
    if (!c.page_ok(from) || !c.page_ok(to)) {
      if (lane == 0) report(kDevBadArgument);
      continue;
    }
    const int64_t size = a.row_bytes / c.head_dim;
    const int64_t src = c.row_offset(from, h, slot & mask) * size, dst = c.row_offset(to, h, (int)(j & mask)) * size;
    for (int i = lane * 16; i < a.row_bytes; i += 512) {
      const uint4 k = *reinterpret_cast<const uint4*>(a.k_pages + src + i);
      const uint4 v = *reinterpret_cast<const uint4*>(a.v_pages + src + i);
      *reinterpret_cast<uint4*>(a.k_pages + dst + i) = k;
      *reinterpret_cast<uint4*>(a.v_pages + dst + i) = v;
    }
  }
}

}  // namespace tq4

using namespace tq4;

extern "C" {

tq4_status tq4_paged_create(const tq4_paged_desc* desc, void* k_pages, void* v_pages,
                            const int32_t* page_table, int device, tq4_paged** out) {
  clear_error();
  if (!desc || !out || !k_pages || !v_pages || !page_table || device < 0) {
    set_error("tq4_paged_create: null description, pages, page table or output, or a negative device");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  *out = nullptr;
  const tq4_paged_desc& d = *desc;
  if (d.dtype != TQ4_F32 && d.dtype != TQ4_F16 && d.dtype != TQ4_BF16) {
    set_error("tq4_paged_create: the pages must be f32, f16 or bf16");
    return TQ4_ERR_UNSUPPORTED;
  }
  if (d.head_dim <= 0 || d.head_dim > 256 || d.head_dim * dtype_size(d.dtype) % 16) {
    set_error("tq4_paged_create: head_dim %d (%s) must take a multiple of 16 bytes and be at most 256", d.head_dim,
              dtype_name(d.dtype));
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (d.page_size <= 0 || (d.page_size & (d.page_size - 1)) != 0) {
    set_error("tq4_paged_create: page_size must be a power of two, got %d", d.page_size);
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (d.kv_heads <= 0 || d.num_pages <= 0 || d.num_pages > INT32_MAX || d.max_seqs <= 0 || d.max_pages <= 0 ||
      (int64_t)d.max_pages * d.page_size > ((int64_t)1 << 30) ||
      d.num_pages > ((int64_t)1 << 32) / d.page_size / d.kv_heads) {
    set_error("tq4_paged_create: kv_heads, num_pages, max_seqs and max_pages must be positive, page numbers below "
              "2^31, a sequence's slots (max_pages * page_size) at most 2^30, the pool's rows (num_pages * kv_heads * page_size) "
              "at most 2^32");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (!aligned16(k_pages) || !aligned16(v_pages) || (reinterpret_cast<uintptr_t>(page_table) & 3)) {
    set_error("tq4_paged_create: the pages must be 16-byte aligned, the page table 4-byte aligned");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  tq4_paged* c = new (std::nothrow) tq4_paged();
  if (!c) {
    set_error("tq4_paged_create: out of host memory");
    return TQ4_ERR_OUT_OF_MEMORY;
  }
  c->desc = d;
  c->device = device;
  c->k_pages = k_pages;
  c->v_pages = v_pages;
  c->page_table = page_table;
  while ((1 << c->page_log2) < d.page_size) ++c->page_log2;
  *out = c;
  return TQ4_OK;
}

tq4_status tq4_paged_destroy(tq4_paged* cache) {
  clear_error();
  delete cache;
  return TQ4_OK;
}

tq4_status tq4_paged_append(const tq4_paged* cache, const void* q, int64_t q_stride, const void* k,
                            int64_t k_stride, const void* v, int64_t v_stride, int heads, int64_t tokens,
                            const int32_t* seq, const int32_t* slot, const int32_t* positions,
                            const tq4_rotary* rotary, void* q_out, void* stream) {
  clear_error();
  if (!cache) {
    set_error("tq4_paged_append: null cache");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  const tq4_paged_desc& d = cache->desc;
  const int64_t rows = (int64_t)heads + 2 * (int64_t)d.kv_heads;
  if (heads < 0 || (heads > 0) != (q != nullptr) || (q && !q_out)) {
    set_error("tq4_paged_append: q and q_out with heads > 0, or neither with heads 0");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (tokens < 0 || tokens > (int64_t)INT32_MAX * (kAppendThreads / 32) / rows) {
    set_error("tq4_paged_append: %lld tokens out of range", (long long)tokens);
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (tokens == 0) return TQ4_OK;
  if (!k || !v || !seq || !slot) {
    set_error("tq4_paged_append: null k, v, seq or slot");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  const int64_t D = d.head_dim;
  if ((q && q_stride < heads * D) || k_stride < d.kv_heads * D || v_stride < d.kv_heads * D) {
    set_error("tq4_paged_append: a token's heads are contiguous: strides of at least heads * head_dim values");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  const int size = dtype_size(d.dtype);
  if (q && overlaps(q, ((tokens - 1) * q_stride + heads * D) * size, q_out, tokens * heads * D * size)) {
    set_error("tq4_paged_append: q_out overlaps q");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  AppendArgs a{};
  a.cache = view_of(*cache);
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_out = q_out;
  a.k_pages = cache->k_pages;
  a.v_pages = cache->v_pages;
  a.seq = seq;
  a.slot = slot;
  a.positions = positions;
  a.tokens = tokens;
  a.heads = heads;
  if (rotary) {
    const tq4_rotary& r = *rotary;
    if (r.pairs < 0 || 2 * (int64_t)r.pairs > D) {
      set_error("tq4_paged_append: %d pairs do not fit head_dim %d", r.pairs, d.head_dim);
      return TQ4_ERR_INVALID_ARGUMENT;
    }
    if (r.pairs > 0 && (!r.cos_table || !r.sin_table || !positions || r.max_pos <= 0 || r.axes < 1 || r.axes > 4)) {
      set_error("tq4_paged_append: a rotation needs cos and sin tables of max_pos > 0 rows, positions and 1 to 4 axes");
      return TQ4_ERR_INVALID_ARGUMENT;
    }
    a.cos_t = r.cos_table;
    a.sin_t = r.sin_table;
    a.max_pos = r.max_pos;
    a.pairs = r.pairs;
    a.axes = r.axes;
    a.interleaved = r.interleaved != 0;
    a.q_w = r.q_w;
    a.k_w = r.k_w;
    a.eps = r.eps;
    for (int i = 0; r.pair_axis && i < r.pairs; ++i) {
      if (r.pair_axis[i] >= r.axes) {
        set_error("tq4_paged_append: pair %d follows axis %d of %d", i, r.pair_axis[i], r.axes);
        return TQ4_ERR_INVALID_ARGUMENT;
      }
      a.pair_axis[i] = r.pair_axis[i];
    }
  }
  DeviceGuard guard(cache->device);
  const int64_t warps = tokens * rows;
  const dim3 grid((unsigned)((warps + kAppendThreads / 32 - 1) / (kAppendThreads / 32)));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (d.dtype) {
    case TQ4_F16: TQ4_CUDA(launch_pdl(append_kernel<__half>, grid, dim3(kAppendThreads), 0, st, a)); break;
    case TQ4_BF16: TQ4_CUDA(launch_pdl(append_kernel<__nv_bfloat16>, grid, dim3(kAppendThreads), 0, st, a)); break;
    default: TQ4_CUDA(launch_pdl(append_kernel<float>, grid, dim3(kAppendThreads), 0, st, a)); break;
  }
  return TQ4_OK;
}

tq4_status tq4_paged_evict(const tq4_paged* cache, const int32_t* lengths, int64_t batch, const float* scores,
                           int64_t keep, int64_t recent, const int32_t* new_table, int32_t new_max_pages,
                           int32_t* new_lengths, int32_t* kept, float* new_scores, int64_t new_score_stride,
                           void* stream) {
  clear_error();
  if (!cache) {
    set_error("tq4_paged_evict: null cache");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  const tq4_paged_desc& d = cache->desc;
  if (batch < 0 || batch > d.max_seqs) {
    set_error("tq4_paged_evict: %lld sequences, the page table has %d", (long long)batch, d.max_seqs);
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (keep < 1 || recent < 0 || recent > keep || keep > (int64_t)new_max_pages * d.page_size || keep > INT32_MAX) {
    set_error("tq4_paged_evict: 0 <= recent <= keep and 1 <= keep <= new_max_pages * page_size, got recent %lld, "
              "keep %lld, %d pages of %d", (long long)recent, (long long)keep, new_max_pages, d.page_size);
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (batch == 0) return TQ4_OK;
  if (!lengths || !scores || !new_table || !new_lengths || !kept) {
    set_error("tq4_paged_evict: null lengths, scores, new_table, new_lengths or kept");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (new_scores && new_score_stride < keep) {
    set_error("tq4_paged_evict: new_score_stride %lld below keep %lld", (long long)new_score_stride, (long long)keep);
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  EvictArgs a{};
  a.cache = view_of(*cache);
  const int64_t rows = batch * d.kv_heads;
  const int64_t table_bytes = (int64_t)d.max_seqs * d.max_pages * 4, score_bytes = rows * a.cache.max_slots * 4;
  const struct { const void* p; int64_t bytes; } in[] = {
      {lengths, batch * 4}, {scores, score_bytes}, {new_table, batch * new_max_pages * 4}, {cache->page_table, table_bytes}};
  const struct { const void* p; int64_t bytes; } outs[] = {
      {new_lengths, batch * 4}, {kept, rows * keep * 4},
      {new_scores, new_scores ? ((rows - 1) * new_score_stride + keep) * 4 : 0}};
  for (const auto& o : outs)
    for (const auto& i : in)
      if (overlaps(o.p, o.bytes, i.p, i.bytes)) {
        set_error("tq4_paged_evict: an output overlaps an input");
        return TQ4_ERR_INVALID_ARGUMENT;
      }
  a.lengths = lengths;
  a.batch = batch;
  a.scores = scores;
  a.keep = keep;
  a.recent = recent;
  a.new_table = new_table;
  a.new_max_pages = new_max_pages;
  a.new_lengths = new_lengths;
  a.kept = kept;
  a.new_scores = new_scores;
  a.new_score_stride = new_score_stride;
  a.k_pages = static_cast<char*>(cache->k_pages);
  a.v_pages = static_cast<char*>(cache->v_pages);
  a.row_bytes = d.head_dim * dtype_size(d.dtype);
  DeviceGuard guard(cache->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows > INT32_MAX) {
    set_error("tq4_paged_evict: too many rows");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  TQ4_CUDA(launch_pdl(evict_select_kernel, dim3((unsigned)rows), dim3(kSelectThreads), 0, st, a));
  const int64_t blocks = (rows * keep + kMoveThreads / 32 - 1) / (kMoveThreads / 32);
  TQ4_CUDA(launch_pdl(evict_move_kernel, dim3((unsigned)std::min<int64_t>(blocks, 148 * 8)), dim3(kMoveThreads), 0, st,
                      a));
  return TQ4_OK;
}

}  // extern "C"
