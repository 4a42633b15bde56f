// Attention of one new token of each sequence over the paged cache (include/tq4_paged.h).
//
// The work is split over the cache's length without the host knowing any length: a sequence's
// slots are cut into units of kUnit, all units of all (sequence, KV head, head tile) rows stand in
// one line, and CTA c of P takes units [c * total / P, (c + 1) * total / P) of it. Each CTA finds
// its place by a prefix sum over the lengths. It folds its part of a row into a running maximum m,
// a sum l of exp2(s - m) and an unnormalised output o (online softmax); a row that lies in one CTA
// is finished there, the parts of others go to the workspace and a second kernel joins them in CTA
// order, so results depend on the lengths alone.
#include "paged.cuh"

namespace tq4 {

constexpr int kUnit = 32;         // slots of a unit: what a warp folds at a time
constexpr int kPartWarps = 4;     // warps of a CTA, taking a row's units in turn
constexpr int kPartThreads = kPartWarps * 32;
constexpr int kHeadTile = 8;      // query heads of a row
constexpr int kPartCtas = 148 * 2;  // two a B200's SM
constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  PagedView cache;
  const void *q, *k_pages, *v_pages;
  int64_t q_stride;
  void* out;
  const int32_t* lengths;
  int64_t batch, window;
  int heads, group, tiles;  // query heads, those of a KV head, tiles of kHeadTile of them
  float scale2;             // scale * log2(e): scores are kept for exp2
  const float* scores;
  float* new_scores;
  // workspace
  float* stats;    // [batch][heads][2]: m, 1 / l of finished rows
  float* parts;    // [kPartCtas][2][kHeadTile][head_dim + 2]: o, m, l
  float* weights;  // [batch][kv_heads][max_slots][group]: scores s * scale2
};

struct Span {
  int64_t lo, hi;  // slots attended to
  __device__ __forceinline__ int64_t units() const { return (hi - lo + kUnit - 1) / kUnit; }
};

__device__ __forceinline__ Span span_of(const AttnArgs& a, int64_t b) {
  const int64_t n = paged_length(a.cache, a.lengths, b);
  return {a.window > 0 && n > a.window ? n - a.window : 0, n};
}

// The line of units: how many there are before sequence `stop` (all of them in *total). Every
// thread of the block calls it; `red` holds one value a thread.
template <int THREADS>
__device__ __forceinline__ int64_t units_before(const AttnArgs& a, int64_t stop, int64_t* red, int64_t* total) {
  int64_t all = 0, before = 0;
  for (int64_t b = threadIdx.x; b < a.batch; b += THREADS) {
    const int64_t u = span_of(a, b).units();
    all += u;
    if (b < stop) before += u;
  }
  for (int off = 16; off > 0; off >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, off);
    before += __shfl_xor_sync(0xffffffffu, before, off);
  }
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    red[2 * warp] = all;
    red[2 * warp + 1] = before;
  }
  __syncthreads();
  all = before = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    all += red[2 * w];
    before += red[2 * w + 1];
  }
  __syncthreads();
  const int64_t rows = (int64_t)a.cache.kv_heads * a.tiles;
  *total = all * rows;
  return before * rows;
}

// The sequence that unit `x` of the line lies in, and the first unit of that sequence.
template <int THREADS>
__device__ __forceinline__ void find_unit(const AttnArgs& a, int64_t x, int64_t* red, int64_t* seq, int64_t* first) {
  // each thread sums a run of sequences, then the run that holds x is walked
  const int64_t rows = (int64_t)a.cache.kv_heads * a.tiles;
  const int64_t per = (a.batch + THREADS - 1) / THREADS;
  const int64_t b0 = min(per * threadIdx.x, a.batch), b1 = min(b0 + per, a.batch);
  int64_t mine = 0;
  for (int64_t b = b0; b < b1; ++b) mine += span_of(a, b).units() * rows;
  int64_t incl = mine;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += y;
  }
  if (lane == 31) red[warp] = incl;
  __syncthreads();
  int64_t at = incl - mine;
  for (int w = 0; w < warp; ++w) at += red[w];
  __syncthreads();
  if (x >= at && x < at + mine) {
    int64_t b = b0;
    for (;; ++b) {
      const int64_t u = span_of(a, b).units() * rows;
      if (x < at + u) break;
      at += u;
    }
    red[0] = b;
    red[1] = at;
  }
  __syncthreads();
  *seq = red[0];
  *first = red[1];
  __syncthreads();
}

__device__ __forceinline__ int64_t first_unit(int64_t total, int cta) { return total * cta / kPartCtas; }
// The CTA whose range holds unit x.
__device__ __forceinline__ int cta_of(int64_t total, int64_t x) { return (int)(((x + 1) * kPartCtas - 1) / total); }

template <typename T> struct Vec16 {
  static constexpr int kN = 16 / sizeof(T);
  T v[kN];
};

// A unit's rows to shared memory: lane i knows the offset and the page of row i. A row behind the
// end (page < 0) may hold anything, NaN too, and becomes zeros.
template <typename T>
__device__ __forceinline__ void load_rows(T* dst, const T* pages, int64_t off, int page, int chunks, int pitch) {
  constexpr int VN = Vec16<T>::kN;
  for (int i = threadIdx.x & 31; i < kUnit * chunks; i += 32) {  // every lane takes `chunks` turns
    const int row = i / chunks, col = i - row * chunks;
    const int64_t ro = __shfl_sync(0xffffffffu, off, row);
    const int rp = __shfl_sync(0xffffffffu, page, row);
    *reinterpret_cast<uint4*>(dst + row * pitch + col * VN) =
        rp >= 0 ? *reinterpret_cast<const uint4*>(pages + ro + col * VN) : make_uint4(0, 0, 0, 0);
  }
}

// T: the cache's type. COLS: groups of 128 output columns (head_dim <= 128 or <= 256).
template <typename T, int COLS>
__global__ void __launch_bounds__(kPartThreads) attention_part_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int VN = Vec16<T>::kN;
  __shared__ int64_t red[2 * kPartWarps];
  __shared__ float qs[kHeadTile][256];
  __shared__ float ps[kPartWarps][kUnit][kHeadTile];
  __shared__ float ml[kPartWarps][kHeadTile][2];
  extern __shared__ __align__(16) char dyn[];
  const PagedView& c = a.cache;
  const int D = c.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int chunks = D / VN;                       // 16-byte chunks of a row
  const int pitch = (chunks | 1) * VN;             // odd in chunks: no bank is met twice by 8 rows
  T* ks = reinterpret_cast<T*>(dyn) + (int64_t)warp * kUnit * pitch;  // the unit's keys, then its values
  float* os = reinterpret_cast<float*>(dyn);       // the warps' outputs, when the row's units are done

  int64_t total, b, b_first;
  units_before<kPartThreads>(a, 0, red, &total);
  int64_t x = first_unit(total, blockIdx.x);
  const int64_t end = first_unit(total, blockIdx.x + 1);
  if (x >= end) return;
  find_unit<kPartThreads>(a, x, red, &b, &b_first);
  const int64_t rows = (int64_t)c.kv_heads * a.tiles;
  Span sp = span_of(a, b);
  int64_t units = sp.units();
  int64_t r = (x - b_first) / units, u0 = (x - b_first) - r * units;

  while (x < end) {
    const int64_t m_units = min(end - x, units - u0);
    const int kvh = (int)(r / a.tiles), g0 = (int)(r % a.tiles) * kHeadTile;
    const int G = min(kHeadTile, a.group - g0), h0 = kvh * a.group + g0;
    __syncthreads();
    for (int i = tid; i < kHeadTile * D; i += kPartThreads) {
      const int g = i / D, d = i - g * D;
      qs[g][d] = g < G ? to_f32(static_cast<const T*>(a.q)[b * a.q_stride + (int64_t)(h0 + g) * D + d]) : 0.f;
    }
    __syncthreads();
    float m[kHeadTile], l[kHeadTile], o[COLS][4][kHeadTile];
#pragma unroll
    for (int g = 0; g < kHeadTile; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int j = 0; j < COLS * 4; ++j) o[j / 4][j % 4][g] = 0.f;
    }
    for (int64_t u = u0 + warp; u < u0 + m_units; u += kPartWarps) {
      const int64_t p = sp.lo + u * kUnit + lane;
      int page = -1;
      if (p < sp.hi) {
        page = c.table[b * c.max_pages + (p >> c.page_log2)];
        if (!c.page_ok(page)) {
          report(kDevBadArgument);
          page = -1;
        }
      }
      const bool valid = page >= 0;
      const int64_t off = c.row_offset(page, kvh, (int)(p & ((1 << c.page_log2) - 1)));
      load_rows<T>(ks, static_cast<const T*>(a.k_pages), off, page, chunks, pitch);
      __syncwarp();
      float s[kHeadTile];
#pragma unroll
      for (int g = 0; g < kHeadTile; ++g) s[g] = 0.f;
      for (int i = 0; i < chunks; ++i) {
        const Vec16<T> kv = *reinterpret_cast<const Vec16<T>*>(ks + lane * pitch + i * VN);
#pragma unroll
        for (int g = 0; g < kHeadTile; ++g)
#pragma unroll
          for (int e = 0; e < VN; ++e) s[g] = fmaf(qs[g][i * VN + e], to_f32(kv.v[e]), s[g]);
      }
      float alpha[kHeadTile];
#pragma unroll
      for (int g = 0; g < kHeadTile; ++g) {
        s[g] = valid ? s[g] * a.scale2 : -INFINITY;
        float mx = s[g];
        for (int of = 16; of > 0; of >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, of));
        mx = fmaxf(mx, m[g]);
        const float base = mx == -INFINITY ? 0.f : mx;  // nothing valid so far: every weight is 0
        alpha[g] = exp2f(m[g] - base);
        m[g] = mx;
        const float e = exp2f(s[g] - base);
        l[g] = l[g] * alpha[g] + e;
        ps[warp][lane][g] = e;
      }
      if (a.new_scores && p < sp.hi) {
        float* w = a.weights + ((b * c.kv_heads + kvh) * c.max_slots + p) * a.group + g0;
#pragma unroll
        for (int g = 0; g < kHeadTile; ++g)
          if (g < G) w[g] = s[g];
      }
      __syncwarp();
      load_rows<T>(ks, static_cast<const T*>(a.v_pages), off, page, chunks, pitch);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < COLS * 4; ++j)
#pragma unroll
        for (int g = 0; g < kHeadTile; ++g) o[j / 4][j % 4][g] *= alpha[g];
      for (int i = 0; i < kUnit; ++i) {
        float pg[kHeadTile];
#pragma unroll
        for (int g = 0; g < kHeadTile; ++g) pg[g] = ps[warp][i][g];
#pragma unroll
        for (int j = 0; j < COLS; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = j * 128 + lane * 4 + e;
            const float vv = d < D ? to_f32(ks[i * pitch + d]) : 0.f;
#pragma unroll
            for (int g = 0; g < kHeadTile; ++g) o[j][e][g] = fmaf(pg[g], vv, o[j][e][g]);
          }
      }
      __syncwarp();
    }
    // the warps' (m, l, o) joined in warp order
#pragma unroll
    for (int g = 0; g < kHeadTile; ++g) {
      for (int of = 16; of > 0; of >>= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], of);
      if (lane == 0) {
        ml[warp][g][0] = m[g];
        ml[warp][g][1] = l[g];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < COLS; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = j * 128 + lane * 4 + e;
        if (d < D)
#pragma unroll
          for (int g = 0; g < kHeadTile; ++g) os[(warp * kHeadTile + g) * D + d] = o[j][e][g];
      }
    __syncthreads();
    const bool whole = m_units == units;
    // a CTA has at most two parts: one of a row that began before it, one of a row that ends behind it
    float* part = a.parts + ((int64_t)blockIdx.x * 2 + (u0 > 0 ? 0 : 1)) * kHeadTile * (D + 2);
    for (int i = tid; i < G * D; i += kPartThreads) {
      const int g = i / D, d = i - g * D;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kPartWarps; ++w) M = fmaxf(M, ml[w][g][0]);
      const float base = M == -INFINITY ? 0.f : M;
      float num = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < kPartWarps; ++w) {
        const float f = exp2f(ml[w][g][0] - base);
        num = fmaf(f, os[(w * kHeadTile + g) * D + d], num);
        den = fmaf(f, ml[w][g][1], den);
      }
      if (whole) {
        const float inv = den > 0.f ? 1.f / den : 0.f;
        static_cast<T*>(a.out)[(b * a.heads + h0 + g) * D + d] = from_f32<T>(den == 0.f ? 0.f : num / den);
        if (d == 0) {
          a.stats[(b * a.heads + h0 + g) * 2] = base;
          a.stats[(b * a.heads + h0 + g) * 2 + 1] = inv;
        }
      } else {
        part[g * (D + 2) + d] = num;
        if (d == 0) {
          part[g * (D + 2) + D] = M;
          part[g * (D + 2) + D + 1] = den;
        }
      }
    }
    x += m_units;
    u0 = 0;
    if (x < end && ++r == rows) {
      r = 0;
      do sp = span_of(a, ++b);
      while ((units = sp.units()) == 0);
    }
  }
}

// One CTA a row: joins the parts of a row that lies in more than one CTA; zeros for a sequence
// without slots.
template <typename T>
__global__ void __launch_bounds__(kPartThreads) attention_join_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ int64_t red[2 * kPartWarps];
  const PagedView& c = a.cache;
  const int D = c.head_dim, tid = threadIdx.x;
  const int64_t rows = (int64_t)c.kv_heads * a.tiles;
  const int64_t b = blockIdx.x / rows, r = blockIdx.x % rows;
  const int kvh = (int)(r / a.tiles), g0 = (int)(r % a.tiles) * kHeadTile;
  const int G = min(kHeadTile, a.group - g0), h0 = kvh * a.group + g0;
  T* out = static_cast<T*>(a.out) + (b * a.heads + h0) * D;
  const int64_t units = span_of(a, b).units();
  if (units == 0) {
    for (int i = tid; i < G * D; i += kPartThreads) out[i] = from_f32<T>(0.f);
    return;
  }
  int64_t total;
  const int64_t x0 = units_before<kPartThreads>(a, b, red, &total) + r * units;
  const int first = cta_of(total, x0), last = cta_of(total, x0 + units - 1);
  if (first == last) return;
  for (int i = tid; i < G * D; i += kPartThreads) {
    const int g = i / D, d = i - g * D;
    float M = -INFINITY;
    for (int k = first; k <= last; ++k) {
      if (first_unit(total, k) == first_unit(total, k + 1)) continue;  // fewer units than CTAs
      M = fmaxf(M, a.parts[((int64_t)(k * 2 + (k == first)) * kHeadTile + g) * (D + 2) + D]);
    }
    const float base = M == -INFINITY ? 0.f : M;
    float num = 0.f, den = 0.f;
    for (int k = first; k <= last; ++k) {
      if (first_unit(total, k) == first_unit(total, k + 1)) continue;
      const float* p = a.parts + ((int64_t)(k * 2 + (k == first)) * kHeadTile + g) * (D + 2);
      const float f = exp2f(p[D] - base);
      num = fmaf(f, p[d], num);
      den = fmaf(f, p[D + 1], den);
    }
    out[i] = from_f32<T>(den == 0.f ? 0.f : num / den);
    if (d == 0) {
      a.stats[(b * a.heads + h0 + g) * 2] = base;
      a.stats[(b * a.heads + h0 + g) * 2 + 1] = den > 0.f ? 1.f / den : 0.f;
    }
  }
}

// new_scores = scores + sum over the group's heads of exp2(s - m) / l; slots before a window keep theirs.
constexpr int kWeightThreads = 256;
__global__ void __launch_bounds__(kWeightThreads) attention_weight_kernel(const __grid_constant__ AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const PagedView& c = a.cache;
  const int64_t rows = a.batch * c.kv_heads;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const int64_t b = row / c.kv_heads;
    const int kvh = (int)(row - b * c.kv_heads);
    const Span sp = span_of(a, b);
    const float* st = a.stats + (b * a.heads + kvh * a.group) * 2;
    for (int64_t p = (int64_t)blockIdx.x * kWeightThreads + threadIdx.x; p < sp.hi; p += (int64_t)gridDim.x * kWeightThreads) {
      float sum = 0.f;
      if (p >= sp.lo) {
        const float* w = a.weights + (row * c.max_slots + p) * a.group;
        for (int g = 0; g < a.group; ++g) sum = fmaf(exp2f(w[g] - st[2 * g]), st[2 * g + 1], sum);
      }
      a.new_scores[row * c.max_slots + p] = a.scores[row * c.max_slots + p] + sum;
    }
  }
}

namespace {

// Offsets of the workspace's parts, in floats, each a multiple of 4.
struct Workspace {
  int64_t parts, weights, floats;
};
Workspace workspace_of(const tq4_paged_desc& d, int heads, int64_t batch, bool with_scores) {
  auto up = [](int64_t n) { return (n + 3) / 4 * 4; };
  Workspace w;
  w.parts = up(batch * heads * 2);
  w.weights = w.parts + up((int64_t)kPartCtas * 2 * kHeadTile * (d.head_dim + 2));
  w.floats = w.weights + (with_scores ? batch * heads * (int64_t)d.max_pages * d.page_size : 0);
  return w;
}

tq4_status check_attention(const tq4_paged* cache, int heads, int64_t batch) {
  if (!cache) {
    set_error("tq4_paged_attention: null cache");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  const tq4_paged_desc& d = cache->desc;
  if (heads <= 0 || heads % d.kv_heads || heads > 65535) {
    set_error("tq4_paged_attention: %d query heads are not a multiple of %d KV heads up to 65535", heads, d.kv_heads);
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (batch < 0 || batch > d.max_seqs) {
    set_error("tq4_paged_attention: %lld sequences, the page table has %d", (long long)batch, d.max_seqs);
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  return TQ4_OK;
}

template <typename T>
tq4_status launch_attention(const AttnArgs& a, cudaStream_t st) {
  const int D = a.cache.head_dim;
  constexpr int VN = Vec16<T>::kN;
  const size_t tiles = (size_t)kPartWarps * kUnit * ((D / VN) | 1) * 16;
  const size_t outs = (size_t)kPartWarps * kHeadTile * D * 4;
  const size_t smem = std::max(tiles, outs);
  const auto part = D <= 128 ? attention_part_kernel<T, 1> : attention_part_kernel<T, 2>;
  static std::atomic<uint64_t> set1{0}, set2{0};
  TQ4_CUDA(set_smem_limit_once(part, 227 * 1024 - 16 * 1024, D <= 128 ? set1 : set2));
  TQ4_CUDA(launch_pdl(part, dim3(kPartCtas), dim3(kPartThreads), smem, st, a));
  const int64_t rows = a.batch * a.cache.kv_heads * a.tiles;
  TQ4_CUDA(launch_pdl(attention_join_kernel<T>, dim3((unsigned)rows), dim3(kPartThreads), 0, st, a));
  return TQ4_OK;
}

}  // namespace

}  // namespace tq4

using namespace tq4;

extern "C" {

tq4_status tq4_paged_attention_workspace(const tq4_paged* cache, int heads, int64_t batch, int with_scores,
                                         int64_t* bytes) {
  clear_error();
  TQ4_TRY(check_attention(cache, heads, batch));
  if (!bytes) {
    set_error("tq4_paged_attention_workspace: null output");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  *bytes = workspace_of(cache->desc, heads, batch, with_scores != 0).floats * 4;
  return TQ4_OK;
}

tq4_status tq4_paged_attention(const tq4_paged* cache, const void* q, int64_t q_stride, int heads,
                               const int32_t* lengths, int64_t batch, float scale, int64_t window,
                               const float* scores, float* new_scores, void* out, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  clear_error();
  TQ4_TRY(check_attention(cache, heads, batch));
  const tq4_paged_desc& d = cache->desc;
  if (batch == 0) return TQ4_OK;
  if (!q || !lengths || !out || !workspace || (scores != nullptr) != (new_scores != nullptr)) {
    set_error("tq4_paged_attention: null q, lengths, out or workspace, or only one of scores and new_scores");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (window < 0 || q_stride < (int64_t)heads * d.head_dim) {
    set_error("tq4_paged_attention: window %lld below 0, or q_stride %lld below heads * head_dim", (long long)window,
              (long long)q_stride);
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  const Workspace ws = workspace_of(d, heads, batch, scores != nullptr);
  if (workspace_bytes < ws.floats * 4 || !aligned16(workspace)) {
    set_error("tq4_paged_attention: the workspace must be 16-byte aligned and hold %lld bytes, got %lld",
              (long long)(ws.floats * 4), (long long)workspace_bytes);
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  AttnArgs a{};
  a.cache = view_of(*cache);
  a.q = q;
  a.k_pages = cache->k_pages;
  a.v_pages = cache->v_pages;
  a.q_stride = q_stride;
  a.out = out;
  a.lengths = lengths;
  a.batch = batch;
  a.window = window;
  a.heads = heads;
  a.group = heads / d.kv_heads;
  a.tiles = (a.group + kHeadTile - 1) / kHeadTile;
  a.scale2 = scale * kLog2e;
  a.scores = scores;
  a.new_scores = new_scores;
  a.stats = static_cast<float*>(workspace);
  a.parts = a.stats + ws.parts;
  a.weights = a.stats + ws.weights;
  if (batch * d.kv_heads * a.tiles > INT32_MAX) {
    set_error("tq4_paged_attention: too many rows");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  DeviceGuard guard(cache->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (d.dtype) {
    case TQ4_F16: TQ4_TRY(launch_attention<__half>(a, st)); break;
    case TQ4_BF16: TQ4_TRY(launch_attention<__nv_bfloat16>(a, st)); break;
    default: TQ4_TRY(launch_attention<float>(a, st)); break;
  }
  if (scores) {
    const int64_t chunks = (a.cache.max_slots + kWeightThreads - 1) / kWeightThreads;
    const dim3 grid((unsigned)std::min<int64_t>(chunks, 64), (unsigned)std::min<int64_t>(batch * d.kv_heads, 65535));
    TQ4_CUDA(launch_pdl(attention_weight_kernel, grid, dim3(kWeightThreads), 0, st, a));
  }
  return TQ4_OK;
}

}  // extern "C"
