// The paged cache's handle, the write of new tokens into it (norm, rotary embedding, pages) and
// eviction by accumulated attention weight (include/tq4_paged.h). Attention is paged_attention.cu.
#include "paged.cuh"
#include "sm100.cuh"

namespace tq4 {

// ---- append -----------------------------------------------------------------------------------
constexpr int kAppendThreads = 256;
constexpr int kAppendMaxPairs = 128;  // head_dim <= 256
constexpr int kAppendSteps = 3;      // rows of a lane, all of whose loads are in flight together

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
  uint32_t pair_axis[kAppendMaxPairs / 16];  // two bits a pair
};

// Where token t goes: whether its numbers are all in range (else the status is set), its page, and the row in it.
struct AppendPlace {
  bool ok;
  int page, in_page;
  int64_t pos[4];
};
__device__ __forceinline__ AppendPlace append_place(const AppendArgs& a, int64_t t, int s, bool tell) {
  const PagedView& c = a.cache;
  AppendPlace p = {};
  const int64_t slot = a.slot[t];
  p.ok = s < c.max_seqs && slot >= 0 && slot < c.max_slots;
  if (a.pairs > 0)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < a.axes) {
        p.pos[i] = a.positions[i * a.tokens + t];
        p.ok = p.ok && p.pos[i] >= 0 && p.pos[i] < a.max_pos;
      }
  p.page = p.ok ? c.table[(int64_t)s * c.max_pages + (slot >> c.page_log2)] : -1;
  p.ok = c.page_ok(p.page);
  if (!p.ok && tell) report(kDevBadArgument);
  p.in_page = (int)(slot & ((1 << c.page_log2) - 1));
  return p;
}

template <int N> __device__ __forceinline__ void load_weights(float (&w)[N], const float* p) {
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    if (N % 4 == 0 && e % 4 == 0) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p + e));
      w[e] = v.x;
      w[e + 1] = v.y;
      w[e + 2] = v.z;
      w[e + 3] = v.w;
    } else if (N % 4 != 0) {
      w[e] = __ldg(p + e);
      w[e + 1] = __ldg(p + e + 1);
    }
  }
}

// Rows in chunks of VE values, 16 bytes or, where views or pairs do not fit those, 8 or 4. A lane has two chunks of a row whose values turn together: chunk u and the one half
// the turned part further, or, interleaved, two neighbours; the unturned rest goes two chunks a lane too. So a
// row is 1 << lpr lanes, and a warp's step takes 32 >> lpr rows of one token; its `steps` share the token's angles,
// in registers. Memory bounds it, and near that the instructions: at 8191 tokens of 36 rows of 128 bf16 values,
// normed, with three axes, a row a warp with one value a load took 218 us, chunks without the loads of all steps
// in flight 75 us, this 45 us (3.4 TB/s; the bytes alone would take 24 us).
// PART: some values are not turned. They do not go through the product, where x * 1 - inf * 0 would make NaN of what
// stands beside an infinity. (Asking each lane also where all are turned takes 47 instead of 46 us there, for more
// spilled registers.)
template <typename T, int VE, bool PART>
__global__ void __launch_bounds__(kAppendThreads, 3) append_rows_kernel(const __grid_constant__ AppendArgs a, int lpr,
                                                                       int steps) {
  pdl_wait();
  pdl_trigger();
  const PagedView& c = a.cache;
  const int lane = threadIdx.x & 31, D = c.head_dim, chunks = D / VE;
  const int sub = lane & ((1 << lpr) - 1), group = lane >> lpr, rows_a_step = 32 >> lpr;
  const int rows = a.heads + 2 * c.kv_heads, turned = a.heads + c.kv_heads;
  const int64_t t = (int64_t)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const int first = (int)blockIdx.y * steps * rows_a_step + group;
  const int half = a.interleaved ? 0 : a.pairs / VE;  // chunks to the partner
  const int ca = sub < half ? sub : 2 * sub, cb = sub < half ? sub + half : ca + 1;
  const bool has_a = ca < chunks, has_b = cb < chunks;

  Packed<T, VE> xa[kAppendSteps], xb[kAppendSteps];
  const T* q = static_cast<const T*>(a.q) + t * a.q_stride;
  const T* kk = static_cast<const T*>(a.k) + t * a.k_stride;
  const T* v = static_cast<const T*>(a.v) + t * a.v_stride;
#pragma unroll
  for (int k = 0; k < kAppendSteps; ++k) {
    const int r = first + k * rows_a_step;
    xa[k].clear();
    xb[k].clear();
    if (k >= steps || r >= rows) continue;
    const T* x = r < a.heads ? q + r * D : r < turned ? kk + (r - a.heads) * D : v + (r - turned) * D;
    if (has_a) xa[k].load(x + ca * VE);
    if (has_b) xb[k].load(x + cb * VE);
  }
  const int s = a.seq[t];
  if (s < 0) return;  // padding
  const AppendPlace place = append_place(a, t, s, lane == 0);
  if (!place.ok) return;
  // the angles of this lane's pairs: VE of them
  alignas(16) float cs[VE], sn[VE];
  const bool turn_a = a.interleaved ? has_a && ca * VE < 2 * a.pairs : sub < half;
  const bool turn_b = a.interleaved ? has_b && cb * VE < 2 * a.pairs : turn_a;
  const int pair0 = a.interleaved ? ca * (VE / 2) : sub * VE;
  const bool angles = first - group < turned;
  // the axes of the lane's pairs; all in one word, since pair0 is a multiple of VE
  const uint32_t axes = angles && pair0 < a.pairs ? a.pair_axis[pair0 / 16] >> (pair0 % 16 * 2) : 0;
  auto table_row = [&](uint32_t axis) -> int64_t {
    return (axis == 0 ? place.pos[0] : axis == 1 ? place.pos[1] : axis == 2 ? place.pos[2] : place.pos[3]) * a.pairs;
  };
  constexpr int kRun = VE < 4 ? VE : 4;  // pairs whose angles come in one load where they follow one axis
#pragma unroll
  for (int e = 0; e < VE; e += kRun) {
    bool on = angles, one = true;  // all of the run turn; all follow one axis
    const uint32_t axis0 = (axes >> (2 * e)) & 3;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      on = on && (!a.interleaved || e + i < VE / 2 ? turn_a : turn_b);
      one = one && ((axes >> (2 * (e + i))) & 3) == axis0;
      cs[e + i] = 1.f;
      sn[e + i] = 0.f;
    }
    if (kRun == 4 && on && one) {
      const int64_t at = table_row(axis0) + pair0 + e;
      *reinterpret_cast<float4*>(cs + e) = __ldg(reinterpret_cast<const float4*>(a.cos_t + at));
      *reinterpret_cast<float4*>(sn + e) = __ldg(reinterpret_cast<const float4*>(a.sin_t + at));
    } else {
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        if (angles && (!a.interleaved || e + i < VE / 2 ? turn_a : turn_b)) {
          const int64_t at = table_row((axes >> (2 * (e + i))) & 3) + pair0 + e + i;
          cs[e + i] = __ldg(a.cos_t + at);
          sn[e + i] = __ldg(a.sin_t + at);
        }
    }
  }
  T* q_out = static_cast<T*>(a.q_out) + t * a.heads * D;
  const int64_t at0 = c.row_offset(place.page, 0, place.in_page), head = (int64_t)D << c.page_log2;
  T* k_out = static_cast<T*>(a.k_pages) + at0;
  T* v_out = static_cast<T*>(a.v_pages) + at0;
  const float inv_d = 1.f / (float)D;
#pragma unroll
  for (int k = 0; k < kAppendSteps; ++k) {
    if (k >= steps) break;
    const int r = first + k * rows_a_step;
    if (r - group < turned) {  // the warp's rows are not all values
      const float* nw = r < a.heads ? a.q_w : a.k_w;
      float fa[VE], fb[VE];
      xa[k].get(fa);  // chunks that are not there are zeros
      xb[k].get(fb);
      if (a.q_w || a.k_w) {  // the same for the warp, whose rows may be of both
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < VE; ++e) ss = fmaf(fb[e], fb[e], fmaf(fa[e], fa[e], ss));
        for (int off = (1 << lpr) / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
        if (nw && r < turned) {
          const float inv = rsqrtf(fmaf(ss, inv_d, a.eps));  // within 2^-22
          float w[VE];
          if (has_a) {
            load_weights<VE>(w, nw + ca * VE);
#pragma unroll
            for (int e = 0; e < VE; ++e) fa[e] = fa[e] * inv * w[e];
          }
          if (has_b) {
            load_weights<VE>(w, nw + cb * VE);
#pragma unroll
            for (int e = 0; e < VE; ++e) fb[e] = fb[e] * inv * w[e];
          }
        }
      }
      if (a.interleaved) {
        if (!PART || turn_a)
#pragma unroll
          for (int e = 0; e < VE / 2; ++e) {
            const float x0 = fa[2 * e], x1 = fa[2 * e + 1];
            fa[2 * e] = x0 * cs[e] - x1 * sn[e];
            fa[2 * e + 1] = x1 * cs[e] + x0 * sn[e];
          }
        if (!PART || turn_b)
#pragma unroll
          for (int e = 0; e < VE / 2; ++e) {
            const float y0 = fb[2 * e], y1 = fb[2 * e + 1];
            fb[2 * e] = y0 * cs[VE / 2 + e] - y1 * sn[VE / 2 + e];
            fb[2 * e + 1] = y1 * cs[VE / 2 + e] + y0 * sn[VE / 2 + e];
          }
      } else if (!PART || turn_a) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float x0 = fa[e], x1 = fb[e];
          fa[e] = x0 * cs[e] - x1 * sn[e];
          fb[e] = x1 * cs[e] + x0 * sn[e];
        }
      }
      // values, and what is neither normed nor turned, stay as they are, bit for bit
      if (r < turned && (!PART || nw || turn_a)) xa[k].set(fa);
      if (r < turned && (!PART || nw || turn_b)) xb[k].set(fb);
    }
    if (r >= rows) continue;
    T* y = r < a.heads ? q_out + r * D : r < turned ? k_out + (r - a.heads) * head : v_out + (r - turned) * head;
    if (has_a) xa[k].store(y + ca * VE);
    if (has_b) xb[k].store(y + cb * VE);
  }
}

// The same for what does not come in such chunks (16-bit views that start off 4 bytes, odd numbers of pairs):
// a warp per row of a token, heads queries, then the keys, then the values.
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
  const AppendPlace place = append_place(a, t, s, lane == 0);
  if (!place.ok) return;
  const int page = place.page, in_page = place.in_page;
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
    const int axis = (a.pair_axis[i / 16] >> (i % 16 * 2)) & 3;
    const int64_t row = (axis == 0 ? place.pos[0] : axis == 1 ? place.pos[1] : axis == 2 ? place.pos[2] : place.pos[3]) * pairs + i;
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
struct EvictArgs {
  PagedView cache;
  const int32_t* lengths;
  int64_t batch;
  const float* scores;
  int keep, recent;
  const int32_t* new_table;
  int32_t new_max_pages;
  int32_t *new_lengths, *kept;
  float* new_scores;
  int64_t new_score_stride;
  char *k_pages, *v_pages;
  int row_bytes, chunk_shift;  // chunk_shift: log2 of a row's 16-byte chunks, or -1
  int key_room;  // keys of its share that a CTA of the selection holds in shared memory
  int move;      // the selection's CTAs move the rows too
};

// A score's place in the order: larger keys for larger scores, -0 as 0, NaN below all.
__device__ __forceinline__ uint32_t score_key(float f) {
  if (f != f) return 0;
  const uint32_t u = __float_as_uint(f + 0.f);  // -0 + 0 = 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float key_score(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

// Moves kept rows [j0, j1) of (sequence b, KV head h), by the block, kMoveRows at a time: threads look the rows'
// places up, then all copy 16-byte chunks, kMoveAtOnce of K and of V in flight a thread.
constexpr int kMoveRows = 64, kMoveAtOnce = 4;
struct MoveRows {
  int64_t from[kMoveRows], to[kMoveRows];  // bytes; from < 0: not to be moved
};
template <int THREADS>
__device__ __forceinline__ void move_rows(const EvictArgs& a, int64_t b, int h, const int32_t* kept, int j0, int j1,
                                          MoveRows& rows) {
  const PagedView& c = a.cache;
  const int mask = (1 << c.page_log2) - 1, chunks = a.row_bytes / 16, size = a.row_bytes / c.head_dim;
  for (int base = j0; base < j1; base += kMoveRows) {
    const int n = min(kMoveRows, j1 - base);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const int j = base + i, slot = kept[j];
      int64_t from = -1, to = 0;
      if (slot >= 0) {
        const int p = c.table[b * c.max_pages + (slot >> c.page_log2)];
        const int q = a.new_table[b * a.new_max_pages + (j >> c.page_log2)];
        if (c.page_ok(p) && c.page_ok(q)) {
          from = c.row_offset(p, h, slot & mask) * size;
          to = c.row_offset(q, h, j & mask) * size;
        } else {
          report(kDevBadArgument);
        }
      }
      rows.from[i] = from;
      rows.to[i] = to;
    }
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < n * chunks; i0 += kMoveAtOnce * THREADS) {
      uint4 k[kMoveAtOnce], v[kMoveAtOnce];
      int64_t to[kMoveAtOnce];
#pragma unroll
      for (int m = 0; m < kMoveAtOnce; ++m) {
        const int i = i0 + m * THREADS, row = a.chunk_shift >= 0 ? i >> a.chunk_shift : i / chunks;
        to[m] = -1;
        if (i < n * chunks && rows.from[row] >= 0) {
          const int at = (i - row * chunks) * 16;
          k[m] = *reinterpret_cast<const uint4*>(a.k_pages + rows.from[row] + at);
          v[m] = *reinterpret_cast<const uint4*>(a.v_pages + rows.from[row] + at);
          to[m] = rows.to[row] + at;
        }
      }
#pragma unroll
      for (int m = 0; m < kMoveAtOnce; ++m)
        if (to[m] >= 0) {
          *reinterpret_cast<uint4*>(a.k_pages + to[m]) = k[m];
          *reinterpret_cast<uint4*>(a.v_pages + to[m]) = v[m];
        }
    }
  }
}

constexpr int kBins = 2048;     // of a pass over 11 bits of the keys
// CTAs of a row at most. Of one row of 131072 slots the whole call (64 kept) takes 28 us with 8 and 35 with 4, of one of
// 340000 slots 119 and 214 us. Where the rows are many 4 are as fast or faster (16 rows of 131072 to 16384: 97.8 and 94.0
// us; 32 rows of 40000 to 64: 34 and 22 us), which the rule in launch_evict does not tell apart; 16 took twice the time
// of 8 for the selection of 16 rows.
constexpr int kMaxCluster = 8;

// One cluster per (sequence, KV head): which slots are kept. A CTA has a share of the candidates, in shared memory
// as keys. The smallest kept key is found by radix selection in three passes of 11, 11 and 10 bits: the
// CTAs count their keys by digit, add up each other's counts through distributed shared memory, and each finds
// the digit for itself. Then the keys above that one and the first of its equals are written out in order: a
// thread has a run of the share, and the counts before it give each key its place. What bounds it is latency: three
// passes and five cluster barriers. 16 rows of 131072 slots take 42 us and 128 rows of up to 8192 take 18 us (the
// scores alone 1.3 us and 0.4 us); with one CTA a row, four passes of 8 bits over global memory and a scan for
// every 1024 slots the first, its move included, took 368 us instead of 96 us.
template <int THREADS>
__global__ void __launch_bounds__(THREADS, 2) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  constexpr int WARPS = THREADS / 32;
  __shared__ __align__(16) int hist[2][kBins];
  __shared__ __align__(16) int sums[kBins];  // of the cluster's counts
  __shared__ int warp_sums[WARPS];
  __shared__ int counts[WARPS][2];  // keys above the edge and equal to it, of each warp
  __shared__ int cta_counts[2];
  __shared__ int s_digit, s_need;
  __shared__ MoveRows rows;
  extern __shared__ uint32_t keys[];
  pdl_wait();
  pdl_trigger();
  const PagedView& c = a.cache;
  const int C = (int)gridDim.x, rank = (int)blockIdx.x;
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  const int64_t b = row / c.kv_heads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool real = b < a.batch;  // the grid's last rows may not be; the same for a cluster
  const int L = real ? (int)paged_length(c, a.lengths, b) : 0;
  const float* sc = a.scores + row * c.max_slots;
  int32_t* kept = a.kept + row * a.keep;
  float* ns = a.new_scores ? a.new_scores + row * a.new_score_stride : nullptr;
  const int stay = min(L, a.keep);
  const int64_t all_threads = (int64_t)C * THREADS, me = (int64_t)rank * THREADS + tid;
  if (real) {
    if (row == b * c.kv_heads && me == 0) a.new_lengths[b] = stay;
    for (int64_t i = stay + me; i < a.keep; i += all_threads) kept[i] = -1;
    if (L <= a.keep) {
      for (int64_t i = me; i < L; i += all_threads) {
        kept[i] = (int32_t)i;
        if (ns) ns[i] = sc[i];
      }
    }
  }
  const int most = a.keep - a.recent;  // kept of the candidates
  if (real && L > a.keep) {            // the same for a cluster
    const int n = L - a.recent;        // candidates, more than `most`
    for (int64_t i = me; i < a.recent; i += all_threads) {
      kept[most + i] = (int32_t)(n + i);
      if (ns) ns[most + i] = sc[n + i];
    }
    // this CTA's share
    const int share = (n + C - 1) / C, lo = min(rank * share, n), m = min(share, n - lo);
    const bool held = m <= a.key_room;
    if (held && most > 0) {
      constexpr int kAtOnce = 8;  // loads in flight
      for (int i0 = tid; i0 < m; i0 += kAtOnce * THREADS) {
        float f[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) f[k] = i0 + k * THREADS < m ? sc[lo + i0 + k * THREADS] : 0.f;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          if (i0 + k * THREADS < m) keys[i0 + k * THREADS] = score_key(f[k]);
      }
    }
    auto key_at = [&](int i) { return held ? keys[i] : score_key(sc[lo + i]); };
    uint32_t edge = 0xffffffffu;
    int need = 0;  // how many of the keys equal to the edge are kept
    if (most > 0) {
      uint32_t prefix = 0;
      need = most;
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        int* mine = hist[pass & 1];
        for (int i = tid; i < kBins; i += THREADS) mine[i] = 0;
        __syncthreads();
        for (int i = tid; i < m; i += THREADS) {
          const uint32_t key = key_at(i);
          if (pass == 0 || ((key ^ prefix) >> (pass == 1 ? 21 : 10)) == 0) atomicAdd(&mine[(key >> shift) & (bins - 1)], 1);
        }
        if (C > 1) cluster_sync_all();
        else __syncthreads();
        const int* all = mine;
        if (C > 1) {
          for (int i = tid * 4; i < kBins; i += THREADS * 4) {
            int4 v = make_int4(0, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r)
              if (r < C) {
                const float4 f = ld_cluster_f32x4(reinterpret_cast<const float*>(&mine[i]), (unsigned)r);
                v.x += __float_as_int(f.x);
                v.y += __float_as_int(f.y);
                v.z += __float_as_int(f.z);
                v.w += __float_as_int(f.w);
              }
            *reinterpret_cast<int4*>(&sums[i]) = v;
          }
          all = sums;
          __syncthreads();
        }
        // bins from the top, a run of them a thread
        constexpr int PER = kBins / THREADS;
        int cnt[PER], sum = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          cnt[k] = all[kBins - 1 - (tid * PER + k)];
          sum += cnt[k];
        }
        int incl = sum;
        for (int off = 1; off < 32; off <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, incl, off);
          if (lane >= off) incl += y;
        }
        if (lane == 31) warp_sums[warp] = incl;
        __syncthreads();
        int above = incl - sum;
        for (int w = 0; w < warp; ++w) above += warp_sums[w];
        if (above < need && above + sum >= need) {
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            if (above < need && above + cnt[k] >= need) {
              s_digit = kBins - 1 - (tid * PER + k);
              s_need = need - above;
            }
            above += cnt[k];
          }
        }
        __syncthreads();
        prefix |= (uint32_t)s_digit << shift;
        need = s_need;
      }
      edge = prefix;
    }
    // A thread has a run of the share, an odd number of keys, so that a warp's reads lie in different banks.
    const int run = ((m + THREADS - 1) / THREADS) | 1, r0 = min(tid * run, m), r1 = most > 0 ? min(r0 + run, m) : r0;
    int above = 0, equal = 0;
    for (int i = r0; i < r1; ++i) {
      const uint32_t key = key_at(i);
      above += key > edge;
      equal += key == edge;
    }
    int above_before = above, equal_before = equal;  // of the CTA's threads up to this one
    for (int off = 1; off < 32; off <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, above_before, off), y = __shfl_up_sync(0xffffffffu, equal_before, off);
      if (lane >= off) {
        above_before += x;
        equal_before += y;
      }
    }
    if (lane == 31) {
      counts[warp][0] = above_before;
      counts[warp][1] = equal_before;
    }
    __syncthreads();
    if (tid == 0) {
      int x = 0, y = 0;
      for (int w = 0; w < WARPS; ++w) {
        x += counts[w][0];
        y += counts[w][1];
      }
      cta_counts[0] = x;
      cta_counts[1] = y;
    }
    if (C > 1) cluster_sync_all();
    else __syncthreads();
    int at = above_before - above, equals = equal_before - equal;  // before this thread's run, of all CTAs
    for (int w = 0; w < warp; ++w) {
      at += counts[w][0];
      equals += counts[w][1];
    }
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r)
      if (r < rank) {
        at += ld_cluster_s32(&cta_counts[0], (unsigned)r);
        equals += ld_cluster_s32(&cta_counts[1], (unsigned)r);
      }
    at += min(equals, need);
    for (int i = r0; i < r1; ++i) {
      const uint32_t key = key_at(i);
      if (key < edge || (key == edge && equals++ >= need)) continue;
      kept[at] = lo + i;
      if (ns) ns[at] = key == 0 || key == 0x80000000u ? sc[lo + i] : key_score(key);  // NaN and zeros have one key each
      ++at;
    }
  }
  // no CTA leaves or goes on while another still reads its counts, or before all slots are written
  if (C > 1) cluster_sync_all();
  else __syncthreads();
  if (a.move && real) {
    const int per = (stay + C - 1) / C;
    move_rows<THREADS>(a, b, (int)(row - b * c.kv_heads), kept, min(rank * per, stay), min((rank + 1) * per, stay), rows);
  }
}

// Moves the kept rows; gridDim.x blocks share a row's. Memory bounds it: 38 us for the 203 MB of 16 sequences of 2047
// kept slots (5.4 TB/s), 48 us for the 268 MB of 2 of 16384 (5.6 TB/s).
constexpr int kMoveThreads = 256;
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictArgs a) {
  __shared__ MoveRows rows;
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  const int64_t b = row / a.cache.kv_heads;
  if (b >= a.batch) return;
  const int stay = a.new_lengths[b];
  const int per = ((stay + (int)gridDim.x - 1) / (int)gridDim.x + 7) / 8 * 8;
  const int j0 = min((int)blockIdx.x * per, stay);
  move_rows<kMoveThreads>(a, b, (int)(row - b * a.cache.kv_heads), a.kept + row * a.keep, j0, min(j0 + per, stay), rows);
}

namespace {

// Up to this many bytes of K and V a CTA, the rows are moved by the selection's own CTAs: a launch less, but only as
// many SMs as it has CTAs (3 rows of 1 MB each took 42 us that way, 7.5 us by a kernel of its own).
constexpr int64_t kMoveInSelection = 160 << 10;

// Whether the rows come in chunks of VE values (*taken), and the launch if so.
template <typename T, int VE>
tq4_status launch_append_rows(const AppendArgs& a, cudaStream_t st, bool* taken) {
  constexpr int kWarps = kAppendThreads / 32;
  const int rows = a.heads + 2 * a.cache.kv_heads, chunks = a.cache.head_dim / VE;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
                       reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.q_out);
  const bool strides = a.q_stride % VE == 0 && a.k_stride % VE == 0 && a.v_stride % VE == 0;
  // angles and norm weights in 16-byte loads
  const bool tables = VE < 4 || (a.pairs % 4 == 0 && aligned16(a.cos_t) && aligned16(a.sin_t) && aligned16(a.q_w) && aligned16(a.k_w));
  const int half = a.interleaved ? 0 : a.pairs / VE, units = half + (chunks - 2 * half + 1) / 2;
  *taken = at % (VE * sizeof(T)) == 0 && strides && tables && (a.interleaved ? 2 * a.pairs : a.pairs) % VE == 0 && units <= 32;
  if (!*taken) return TQ4_OK;
  int lpr = 0;
  while ((1 << lpr) < units) ++lpr;
  // few tokens are spread over the SMs
  const int all = (rows + (32 >> lpr) - 1) / (32 >> lpr);
  const int most = (int)std::min<int64_t>(kAppendSteps, std::max<int64_t>(1, a.tokens * all / (148 * 16)));
  const int warps = (all + most - 1) / most, steps = (all + warps - 1) / warps;
  const dim3 grid((unsigned)((a.tokens + kWarps - 1) / kWarps), (unsigned)warps);
  const auto kern = 2 * a.pairs < a.cache.head_dim ? append_rows_kernel<T, VE, true> : append_rows_kernel<T, VE, false>;
  TQ4_CUDA(launch_pdl(kern, grid, dim3(kAppendThreads), 0, st, a, lpr, steps));
  return TQ4_OK;
}

template <typename T>
tq4_status launch_append(const AppendArgs& a, cudaStream_t st) {
  constexpr int kWarps = kAppendThreads / 32;
  const int rows = a.heads + 2 * a.cache.kv_heads;
  bool taken = false;
  if constexpr (sizeof(T) == 2) {
    TQ4_TRY((launch_append_rows<T, 8>(a, st, &taken)));
    if (taken) return TQ4_OK;
  }
  TQ4_TRY((launch_append_rows<T, 4>(a, st, &taken)));
  if (taken) return TQ4_OK;
  TQ4_TRY((launch_append_rows<T, 2>(a, st, &taken)));
  if (taken) return TQ4_OK;
  const int64_t blocks = (a.tokens * rows + kWarps - 1) / kWarps;
  TQ4_CUDA(launch_pdl(append_kernel<T>, dim3((unsigned)blocks), dim3(kAppendThreads), 0, st, a));
  return TQ4_OK;
}

template <int THREADS>
tq4_status launch_select(const EvictArgs& a, dim3 grid, size_t smem, cudaStream_t st) {
  static std::atomic<uint64_t> set{0};  // per device, per instantiation
  TQ4_CUDA(set_smem_limit_once(evict_select_kernel<THREADS>, 200 * 1024, set));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = grid.x;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  TQ4_CUDA(cudaLaunchKernelEx(&cfg, evict_select_kernel<THREADS>, a));
  return TQ4_OK;
}

tq4_status launch_evict(EvictArgs& a, int64_t rows, cudaStream_t st) {
  const int64_t slots = a.cache.max_slots;
  // a CTA has 8192 candidates at most where the cluster's size and the SMs allow it
  int cluster = 1;
  while (cluster < kMaxCluster && slots > (int64_t)cluster * 8192 && rows * cluster * 2 <= 148 * 2) cluster *= 2;
  const int64_t share = (slots + cluster - 1) / cluster;
  a.key_room = (int)std::min<int64_t>(share, 40 * 1024);
  const unsigned y = (unsigned)std::min<int64_t>(rows, 65535), z = (unsigned)((rows + y - 1) / y);
  a.move = (int64_t)a.keep * a.row_bytes * 2 <= cluster * kMoveInSelection;
  const bool small = share <= 2048;
  const size_t smem = (size_t)a.key_room * 4;
  if (small) TQ4_TRY(launch_select<256>(a, dim3(cluster, y, z), smem, st));
  else TQ4_TRY(launch_select<512>(a, dim3(cluster, y, z), smem, st));
  if (a.move) return TQ4_OK;
  const int64_t tiles = (a.keep + kMoveRows - 1) / kMoveRows;
  const unsigned blocks = (unsigned)std::min<int64_t>(tiles, std::max<int64_t>(1, 148 * 16 / rows));
  TQ4_CUDA(launch_pdl(evict_move_kernel, dim3(blocks, y, z), dim3(kMoveThreads), 0, st, a));
  return TQ4_OK;
}

}  // namespace

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
  if (d.kv_heads <= 0 || d.kv_heads > 16384 || d.num_pages <= 0 || d.num_pages > INT32_MAX || d.max_seqs <= 0 || d.max_pages <= 0 ||
      (int64_t)d.max_pages * d.page_size > ((int64_t)1 << 30) ||
      d.num_pages > ((int64_t)1 << 32) / d.page_size / d.kv_heads) {
    set_error("tq4_paged_create: kv_heads (to 16384), num_pages, max_seqs and max_pages must be positive, page numbers below "
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
  // (an empty tensor's address may be null, queries or not)
  if (heads < 0 || heads > 65535 || (tokens != 0 && ((heads > 0) != (q != nullptr) || (q && !q_out)))) {
    set_error("tq4_paged_append: q and q_out with 1 to 65535 heads, or neither with heads 0");
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
  auto bytes = [&](int64_t stride, int64_t n) { return ((tokens - 1) * stride + n * D) * size; };
  if (q && (overlaps(q, bytes(q_stride, heads), q_out, tokens * heads * D * size) ||
            overlaps(k, bytes(k_stride, d.kv_heads), q_out, tokens * heads * D * size) ||
            overlaps(v, bytes(v_stride, d.kv_heads), q_out, tokens * heads * D * size))) {
    set_error("tq4_paged_append: q_out overlaps q, k or v");
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
      a.pair_axis[i / 16] |= (uint32_t)r.pair_axis[i] << (i % 16 * 2);
    }
  }
  DeviceGuard guard(cache->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (d.dtype) {
    case TQ4_F16: return launch_append<__half>(a, st);
    case TQ4_BF16: return launch_append<__nv_bfloat16>(a, st);
    default: return launch_append<float>(a, st);
  }
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
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < i; ++j)
      if (overlaps(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) {
        set_error("tq4_paged_evict: two outputs overlap");
        return TQ4_ERR_INVALID_ARGUMENT;
      }
  a.lengths = lengths;
  a.batch = batch;
  a.scores = scores;
  a.keep = (int)keep;
  a.recent = (int)recent;
  a.new_table = new_table;
  a.new_max_pages = new_max_pages;
  a.new_lengths = new_lengths;
  a.kept = kept;
  a.new_scores = new_scores;
  a.new_score_stride = new_score_stride;
  a.k_pages = static_cast<char*>(cache->k_pages);
  a.v_pages = static_cast<char*>(cache->v_pages);
  a.row_bytes = d.head_dim * dtype_size(d.dtype);
  a.chunk_shift = -1;
  for (int i = 0; i < 8; ++i)
    if (a.row_bytes == 16 << i) a.chunk_shift = i;
  if (rows > (int64_t)65535 * 65535) {
    set_error("tq4_paged_evict: too many rows of sequences and KV heads");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  DeviceGuard guard(cache->device);
  return launch_evict(a, rows, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
