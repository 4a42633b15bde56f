// Attention of one new token of each sequence over the paged cache (include/tq4_paged.h).
//
// A cache row is read once and used by the query heads of its KV head alone, so memory bounds this:
// 2 * head_dim values a slot and KV head. The kernels are built around keeping loads in flight.
//
// The work is split over the cache's length without the host knowing any length: a sequence's
// slots are cut into units of U (8 to 32, a warp's step), all units of all (sequence, KV head, head
// tile) rows stand in one line, and CTA c of P takes units [c * total / P, (c + 1) * total / P) of
// it; each CTA finds its place by a prefix sum over the lengths. Its four warps take the units in
// turn, each through a ring of kStages units of its own that cp.async fills, also across the rows'
// borders, so that the loads never wait for the arithmetic. A warp folds its units into a running
// maximum m, a sum l of exp2(s - m) and an unnormalised output o (online softmax); where a row ends
// the warps' (m, l, o) are joined in shared memory. A row that lies in one CTA is finished there, the
// parts of others go to the workspace and a second kernel joins them in CTA order, so results depend
// on the lengths alone.
#include "paged.cuh"

namespace tq4 {

constexpr int kPartWarps = 4;
constexpr int kPartThreads = kPartWarps * 32;
constexpr int kStages = 3;
constexpr int kSms = 148;  // of a B200; only a grid's size, no CTA waits for another
constexpr int kMaxCtas = kSms * 2;
constexpr int kMaxTile = 16;  // query heads of a row at most
constexpr float kLog2e = 1.4426950408889634f;

// What a part CTA leaves for the second kernel: where its units begin, and the row that began in an
// earlier CTA and ends in this one, if there is one.
struct PartInfo {
  int64_t total;                // units in the line
  int64_t seq_first;            // first unit of sequence b
  int32_t b, r, u0;             // sequence, row and unit of the CTA's first; b < 0: it has none
  int32_t end_b, end_r, first;  // the row that ends here and the CTA it began in; end_b < 0: none
};

struct AttnArgs {
  PagedView cache;
  const void *q, *k_pages, *v_pages;
  int64_t q_stride;
  void* out;
  const int32_t* lengths;
  int64_t batch, window;
  int heads, group;  // query heads, those of a KV head
  int tile, tiles;   // heads of a row, and rows of a KV head
  int unit, unit_log2, ctas;  // slots of a unit; CTAs the line is cut for
  int q_even;        // q's heads are 4-byte aligned
  float scale2;      // scale * log2(e): scores are kept for exp2
  const float* scores;
  float* new_scores;
  // workspace
  PartInfo* info;  // [kMaxCtas]
  float* stats;    // [batch][heads][2]: m, 1 / l of rows that lie in one CTA
  float* ml;       // [kMaxCtas][2][kMaxTile][2]: m, l of the parts of others
  float* parts;    // [kMaxCtas][2][tile][head_dim]: their o
  float* weights;  // [batch][kv_heads][max_slots][group]: scores times scale2
};

struct Span {
  int lo, hi;  // slots attended to
};

__device__ __forceinline__ Span span_of(const AttnArgs& a, int64_t b) {
  const int64_t n = paged_length(a.cache, a.lengths, b);
  return {(int)(a.window > 0 && n > a.window ? n - a.window : 0), (int)n};
}
// Units start at multiples of their size, so that one lies in one page where pages are no smaller; the
// first of a window and the last may be partly outside the span.
__device__ __forceinline__ int units_of(const AttnArgs& a, Span s) {
  return (int)(((unsigned)s.hi + a.unit - 1) >> a.unit_log2) - (s.lo >> a.unit_log2);
}
// First slot of unit u.
__device__ __forceinline__ int unit_slot(const AttnArgs& a, Span s, int u) {
  return ((s.lo >> a.unit_log2) + u) << a.unit_log2;
}

// CTAs that take part: each warp of them gets a unit at least, so a short line is not spread thin.
__device__ __forceinline__ int active_ctas(const AttnArgs& a, int64_t total) {
  return (int)min((int64_t)a.ctas, (total + kPartWarps - 1) / kPartWarps);
}
__device__ __forceinline__ int64_t first_unit(int64_t total, int ctas, int cta) { return total * cta / ctas; }
// The CTA whose range holds unit x.
__device__ __forceinline__ int cta_of(int64_t total, int ctas, int64_t x) {
  return (int)(((x + 1) * ctas - 1) / total);
}

// The line's length, and of unit first_unit(blockIdx.x): its sequence and that sequence's first
// unit. Each thread sums a run of sequences; the run that holds the unit is walked.
struct Place {
  int64_t total, begin, end, seq_first;
  int b;
};
__device__ __forceinline__ Place find_place(const AttnArgs& a, int64_t* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t rows = (int64_t)a.cache.kv_heads * a.tiles;
  const int per = (int)((a.batch + kPartThreads - 1) / kPartThreads);
  const int b0 = (int)min((int64_t)per * tid, a.batch), b1 = (int)min((int64_t)b0 + per, a.batch);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += units_of(a, span_of(a, b)) * rows;
  int64_t incl = mine;
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += y;
  }
  if (lane == 31) red[warp] = incl;
  __syncthreads();
  Place p;
  p.total = 0;
  int64_t at = incl - mine;
  for (int w = 0; w < kPartWarps; ++w) {
    if (w == warp) at += p.total;
    p.total += red[w];
  }
  const int ctas = active_ctas(a, p.total);
  p.begin = p.end = 0;
  p.seq_first = 0;
  p.b = -1;
  if ((int)blockIdx.x >= ctas) return p;  // the same for every thread
  p.begin = first_unit(p.total, ctas, blockIdx.x);
  p.end = first_unit(p.total, ctas, blockIdx.x + 1);
  __syncthreads();
  if (p.begin >= at && p.begin < at + mine) {
    int b = b0;
    for (;; ++b) {
      const int64_t u = units_of(a, span_of(a, b)) * rows;
      if (p.begin < at + u) break;
      at += u;
    }
    red[0] = b;
    red[1] = at;
  }
  __syncthreads();
  p.b = (int)red[0];
  p.seq_first = red[1];
  return p;
}

// A place in the line, stepped forward.
struct Cursor {
  int b, r, u, units;
  Span span;
  __device__ __forceinline__ void set(const AttnArgs& a, int b_, int64_t off) {
    b = b_;
    span = span_of(a, b);
    units = units_of(a, span);
    r = (int)(off / units);
    u = (int)(off - (int64_t)r * units);
  }
  // `n` units on; the caller knows that the line goes that far.
  __device__ __forceinline__ void step(const AttnArgs& a, int rows, int n) {
    u += n;
    while (u >= units) {
      u -= units;
      if (++r == rows) {
        r = 0;
        do span = span_of(a, ++b);
        while ((units = units_of(a, span)) == 0);
      }
    }
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  const int n = take ? 16 : 0;  // what is not taken becomes zeros, and its address is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// 2^x, within 2^-22 of it; 0 for -inf.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// d += a b, 16 x 8 x 16
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Rows in shared memory: an odd number of 16-byte chunks apart, so that the 8 rows of an ldmatrix or
// of a quarter warp's 16-byte loads lie in different banks; 16-bit rows have whole 16-value steps.
template <typename T> __host__ __device__ constexpr int row_chunks(int head_dim) {
  const int values = sizeof(T) == 2 ? (head_dim + 15) / 16 * 16 : head_dim;
  return (values * (int)sizeof(T) / 16) | 1;
}

// ---- 16-bit caches: tensor cores ----------------------------------------------------------------
// A unit is folded with keys and values as the large operand: S^T = K Q^T has 16 slots a row block
// and 8 heads a column block, O^T = V^T P^T 16 columns of the head and 8 heads, so a group of up to 8
// heads fills the instruction; K comes by ldmatrix, V by its transposing form, and the weights turn
// from S^T's layout to P^T's by transposing 8 x 8 blocks between registers. The weights are rounded
// to the cache's type, once, for that product; l sums them unrounded. For f16 they are scaled by
// 2^15 (kBias), so that weights down to 2^-29 of the largest keep f16's full precision.
template <typename T, int DT, int TILE>
struct MmaFold {
  static constexpr int U = DT == 64 ? 32 : 16;
  static constexpr int NT = TILE / 8;  // column blocks of heads
  static constexpr int KS = DT / 16;   // 16-value steps of a row
  static constexpr float kBias = std::is_same_v<T, __half> ? 15.f : 0.f;
  uint32_t qf[NT][KS][2];
  float o[NT][KS][4];
  float m[NT][2], l[NT][2];  // heads 2 * (lane % 4) + {0, 1} of each block

  __device__ __forceinline__ void begin(const AttnArgs& a, int64_t b, int h0, int G, float*, int) {
    const int lane = threadIdx.x & 31, D = a.cache.head_dim;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int g = n * 8 + (lane >> 2);
      const T* src = static_cast<const T*>(a.q) + b * a.q_stride + (int64_t)(h0 + g) * D;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int d = k * 16 + i * 8 + (lane & 3) * 2;
          uint32_t v = 0;
          if (g < G && d < D) {
            if (a.q_even) {
              v = *reinterpret_cast<const uint32_t*>(src + d);
            } else {
              const uint16_t* s = reinterpret_cast<const uint16_t*>(src + d);
              v = s[0] | ((uint32_t)s[1] << 16);
            }
          }
          qf[n][k][i] = v;
        }
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][k][i] = 0.f;
    }
  }

  // One unit: keys at `ks`, values behind them; bit i of `valid`: slot i counts.
  // w, if not null: where the scores of slots `from` to `to` go.
  template <bool WHOLE>
  __device__ __forceinline__ void fold(const AttnArgs& a, const char* ks, uint32_t valid, int row_bytes_, int steps,
                                       float* w, int from, int to, int G, float*, const float*) {
    const int row_bytes = WHOLE ? row_chunks<T>(DT) * 16 : row_bytes_;
    const int lane = threadIdx.x & 31;
    const uint32_t kaddr = smem_u32(ks) + (lane & 15) * row_bytes + (lane >> 4) * 16;
    const uint32_t vaddr = smem_u32(ks) + (U + (lane & 7) + (lane >> 4) * 8) * row_bytes + ((lane >> 3) & 1) * 16;
    float s[U / 16][NT][4];
#pragma unroll
    for (int t = 0; t < U / 16; ++t) {
      float s2[NT][4];  // a second sum halves the chain of dependent products
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][n][i] = s2[n][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
        if (WHOLE || k < steps) {
          uint32_t kf[4];
          ldmatrix_x4(kf, kaddr + t * 16 * row_bytes + k * 32);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<T>(k & 1 ? s2[n] : s[t][n], kf, qf[n][k][0], qf[n][k][1]);
        }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int slot = t * 16 + (lane >> 2) + (i >> 1) * 8;
          s[t][n][i] = (valid >> slot) & 1 ? (s[t][n][i] + s2[n][i]) * a.scale2 : -INFINITY;
          const int g = n * 8 + (lane & 3) * 2 + (i & 1);
          if (w && slot >= from && slot < to && g < G) w[(int64_t)slot * a.group + g] = s[t][n][i];
        }
    }
    uint32_t pf[U / 16][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float mx[2], f[2];
      bool moved = false;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mx[j] = fmaxf(s[0][n][j], s[0][n][j + 2]);
#pragma unroll
        for (int t = 1; t < U / 16; ++t) mx[j] = fmaxf(mx[j], fmaxf(s[t][n][j], s[t][n][j + 2]));
        for (int off = 4; off < 32; off <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], off));
        mx[j] = fmaxf(m[n][j], mx[j] - kBias);
        f[j] = mx[j] == -INFINITY ? 0.f : mx[j];  // nothing counted so far: every weight is 0
        moved = moved || mx[j] != m[n][j];
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float alpha = ex2(m[n][j] - f[j]);
          l[n][j] *= alpha;
          m[n][j] = mx[j];
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            o[n][k][j] *= alpha;
            o[n][k][j + 2] *= alpha;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < U / 16; ++t) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = ex2(s[t][n][i] - f[i & 1]);
          l[n][i & 1] += p[i];
        }
        pf[t][n][0] = transpose8x8(pack2<T>(p[0], p[1]));
        pf[t][n][1] = transpose8x8(pack2<T>(p[2], p[3]));
      }
    }
#pragma unroll
    for (int t = 0; t < U / 16; ++t)
#pragma unroll
      for (int k = 0; k < KS; ++k)
        if (WHOLE || k < steps) {
          uint32_t vf[4];
          ldmatrix_x4_trans(vf, vaddr + t * 16 * row_bytes + k * 32);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<T>(o[n][k], vf, pf[t][n][0], pf[t][n][1]);
        }
  }

  // o to os[TILE][D], m and l to ml[TILE][2].
  __device__ __forceinline__ void end(float* os, float* ml, int D) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        for (int off = 4; off < 32; off <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], off);
        const int g = n * 8 + (lane & 3) * 2 + j;
        if (lane < 4) {
          ml[2 * g] = m[n][j];
          ml[2 * g + 1] = l[n][j];
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const int d = k * 16 + (lane >> 2);
          if (d < D) os[g * D + d] = o[n][k][j];
          if (d + 8 < D) os[g * D + d + 8] = o[n][k][j + 2];
        }
      }
    }
  }
};

// ---- f32 caches: FMA ------------------------------------------------------------------------------
// Scores: a lane takes 4 slots (lane % (U / 4)) and every (128 / U)-th 16-byte chunk of their rows, so a
// chunk of q read from shared memory serves 4 slots and one of K all heads; the lanes' sums are
// then added by halving: each step a lane keeps half of its sums and gives the other half away, 4 *
// TILE values in log steps. Outputs: a lane has 4 columns of the head (lane * 4, and 128 further),
// for all heads.
template <int DT, int TILE>
struct FmaFold {
  static constexpr int U = DT == 64 ? 16 : 8;
  static constexpr int PG = U / 4;         // groups of 4 slots
  static constexpr int SLICES = 32 / PG;   // lanes that share a slot's row
  static constexpr int KJ = (DT / 4 + SLICES - 1) / SLICES;  // chunks of a lane
  static constexpr int COLS = DT <= 128 ? 1 : 2;
  static constexpr int N = 4 * TILE;
  static constexpr int STEPS = PG == 2 ? 4 : 3;
  static constexpr int LEFT = (N >> STEPS) > 0 ? (N >> STEPS) : 1;             // sums a lane ends with
  static constexpr int COPIES = (1 << STEPS) > N ? (1 << STEPS) / N : 1;       // lanes that end with the same
  float o[COLS][4][TILE];
  float m, l;  // of the head that this lane's sums belong to
  int idx;     // they are numbers idx, idx + 1, ...: head idx / 4, slots idx % 4

  __device__ __forceinline__ void begin(const AttnArgs& a, int64_t b, int h0, int G, float* qs, int) {
    const int lane = threadIdx.x & 31, D = a.cache.head_dim;
    for (int i = threadIdx.x; i < TILE * D; i += kPartThreads) {
      const int g = i / D;
      qs[i] = g < G ? static_cast<const float*>(a.q)[b * a.q_stride + (int64_t)h0 * D + i] : 0.f;
    }
    __syncthreads();
    m = -INFINITY;
    l = 0.f;
    idx = 0;
    int n = N;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
      if (n > 1) {
        n /= 2;
        if (lane & (16 >> s)) idx += n;
      }
#pragma unroll
    for (int g = 0; g < TILE; ++g)
#pragma unroll
      for (int j = 0; j < COLS * 4; ++j) o[j / 4][j % 4][g] = 0.f;
  }

  template <bool WHOLE>
  __device__ __forceinline__ void fold(const AttnArgs& a, const char* ks, uint32_t valid, int row_bytes_, int chunks_,
                                       float* w, int from, int to, int G, float* ps, const float* qs) {
    const int lane = threadIdx.x & 31, D = WHOLE ? DT : a.cache.head_dim;
    const int chunks = WHOLE ? DT / 4 : chunks_, row_bytes = WHOLE ? row_chunks<float>(DT) * 16 : row_bytes_;
    const int pg = lane & (PG - 1), slice = lane / PG;
    float v[N];  // [head][4 slots]
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      const int c = slice + j * SLICES;
      if (c < chunks) {
        float4 kv[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) kv[k] = *reinterpret_cast<const float4*>(ks + (pg * 4 + k) * row_bytes + c * 16);
#pragma unroll
        for (int g = 0; g < TILE; ++g) {
          const float4 qv = *reinterpret_cast<const float4*>(qs + g * D + c * 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float& x = v[g * 4 + k];
            x = fmaf(qv.x, kv[k].x, x);
            x = fmaf(qv.y, kv[k].y, x);
            x = fmaf(qv.z, kv[k].z, x);
            x = fmaf(qv.w, kv[k].w, x);
          }
        }
      }
    }
    halve<N, 0>(v, lane);
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < LEFT; ++i) {
      const int slot = pg * 4 + ((idx + i) & 3), g = idx >> 2;
      v[i] = (valid >> slot) & 1 ? v[i] * a.scale2 : -INFINITY;
      mx = fmaxf(mx, v[i]);
      if (w && slot >= from && slot < to && g < G) w[(int64_t)slot * a.group + g] = v[i];
    }
#pragma unroll
    for (int off = 16 / TILE; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    mx = fmaxf(m, mx);
    const float f = mx == -INFINITY ? 0.f : mx;
    const bool moved = __any_sync(0xffffffffu, mx != m);
    const float alpha = ex2(m - f);
    l *= alpha;
    m = mx;
#pragma unroll
    for (int i = 0; i < LEFT; ++i) {
      const float p = ex2(v[i] - f);
      l += p;
      ps[(pg * 4 + ((idx + i) & 3)) * TILE + (idx >> 2)] = p;
    }
    if (moved) {
#pragma unroll
      for (int g = 0; g < TILE; ++g) {
        const float f_g = __shfl_sync(0xffffffffu, alpha, g * (32 / TILE));
#pragma unroll
        for (int j = 0; j < COLS * 4; ++j) o[j / 4][j % 4][g] *= f_g;
      }
    }
    __syncwarp();
    const char* vs = ks + U * row_bytes;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      alignas(16) float pg_[TILE];
      if constexpr (TILE >= 4) {
#pragma unroll
        for (int g = 0; g < TILE; g += 4)
          *reinterpret_cast<float4*>(pg_ + g) = *reinterpret_cast<const float4*>(ps + i * TILE + g);
      } else {
#pragma unroll
        for (int g = 0; g < TILE; ++g) pg_[g] = ps[i * TILE + g];
      }
#pragma unroll
      for (int j = 0; j < COLS; ++j)
        if (lane + j * 32 < chunks) {
          const float4 x = *reinterpret_cast<const float4*>(vs + i * row_bytes + (lane + j * 32) * 16);
#pragma unroll
          for (int g = 0; g < TILE; ++g) {
            o[j][0][g] = fmaf(pg_[g], x.x, o[j][0][g]);
            o[j][1][g] = fmaf(pg_[g], x.y, o[j][1][g]);
            o[j][2][g] = fmaf(pg_[g], x.z, o[j][2][g]);
            o[j][3][g] = fmaf(pg_[g], x.w, o[j][3][g]);
          }
        }
    }
  }

  // Adds M sums over the lanes that differ in bit 4 - S and the bits below it down to PG's.
  template <int M, int S>
  static __device__ __forceinline__ void halve(float* v, int lane) {
    if constexpr (S < STEPS) {
      constexpr int bit = 16 >> S;
      if constexpr (M > 1) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < M / 2; ++i) {
          const float give = up ? v[i] : v[i + M / 2], keep = up ? v[i + M / 2] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
        }
        halve<M / 2, S + 1>(v, lane);
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], bit);
        halve<1, S + 1>(v, lane);
      }
    }
  }

  __device__ __forceinline__ void end(float* os, float* ml, int D) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int off = 16 / TILE; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    if ((lane & (32 / TILE - 1)) == 0) {
      ml[2 * (idx >> 2)] = m;
      ml[2 * (idx >> 2) + 1] = l * (1.f / COPIES);
    }
#pragma unroll
    for (int j = 0; j < COLS; ++j)
      if ((lane + j * 32) * 4 < D)
#pragma unroll
        for (int g = 0; g < TILE; ++g)
          *reinterpret_cast<float4*>(os + g * D + (lane + j * 32) * 4) =
              make_float4(o[j][0][g], o[j][1][g], o[j][2][g], o[j][3][g]);
  }
};

template <typename T, int DT, int TILE>
using FoldOf = std::conditional_t<sizeof(T) == 4, FmaFold<DT, TILE>, MmaFold<T, DT, TILE>>;

// Dynamic shared memory: the rings, then for f32 the queries and each warp's weights.
template <typename T, int DT, int TILE> constexpr int part_smem(int head_dim) {
  constexpr int U = FoldOf<T, DT, TILE>::U;
  return kPartWarps * kStages * 2 * U * row_chunks<T>(head_dim) * 16 +
         (sizeof(T) == 4 ? TILE * head_dim * 4 + kPartWarps * U * TILE * 4 : 0);
}

// WHOLE: head_dim is DT and a page holds whole units. Then a unit's keys are one run of memory, as are its
// values: one page lookup and constant offsets instead of one row address for each chunk (the loads of
// a unit take 30 instructions a lane instead of 300).
template <typename T, int DT, int TILE, bool WHOLE>
__global__ void __launch_bounds__(kPartThreads, DT <= 128 ? 2 : 1)
    attention_part_kernel(const __grid_constant__ AttnArgs a) {
  using Fold = FoldOf<T, DT, TILE>;
  constexpr int U = Fold::U;
  constexpr int VN = 16 / sizeof(T);
  __shared__ int64_t red[2 * kPartWarps];
  __shared__ float ml[kPartWarps][TILE][2];
  __shared__ uint32_t valid_of[kPartWarps][kStages];
  __shared__ int free_of[kPartWarps];
  extern __shared__ __align__(16) char dyn[];
  pdl_wait();
  pdl_trigger();
  const PagedView& c = a.cache;
  const int D = WHOLE ? DT : c.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int chunks = D / VN, row_bytes = row_chunks<T>(D) * 16;
  const int slot_bytes = 2 * U * row_bytes;
  char* ring = dyn + warp * kStages * slot_bytes;
  float* qs = reinterpret_cast<float*>(dyn + kPartWarps * kStages * slot_bytes);
  float* ps = qs + TILE * D + warp * U * TILE;
  const int rows = c.kv_heads * a.tiles;

  // sequences without slots give zeros
  for (int64_t b = blockIdx.x; b < a.batch; b += gridDim.x)
    if (span_of(a, b).hi == 0)
      for (int i = tid; i < a.heads * D; i += kPartThreads) static_cast<T*>(a.out)[b * a.heads * D + i] = from_f32<T>(0.f);

  const Place place = find_place(a, red);
  PartInfo info = {place.total, place.seq_first, -1, 0, 0, -1, 0, 0};
  if (place.b < 0) {
    if (tid == 0) a.info[blockIdx.x] = info;
    return;
  }
  const int ctas = active_ctas(a, place.total);
  Cursor at;  // the row being folded
  at.set(a, place.b, place.begin - place.seq_first);
  info.b = at.b;
  info.r = at.r;
  info.u0 = at.u;

  // 16-bit rows of an odd number of chunks: their last 16-value step reads one more, kept at zero
  auto zero_tails = [&](char* rows_at, int n) {
    if (sizeof(T) == 2 && (chunks & 1))
      for (int i = lane; i < n; i += 32)
        *reinterpret_cast<uint4*>(rows_at + i * row_bytes + chunks * 16) = make_uint4(0, 0, 0, 0);
  };
  zero_tails(ring, kStages * 2 * U);

  // This warp's loads: units begin + warp, + 4, ... A unit's page is looked up one unit ahead of its
  // use: by lane i for slot i, or for all of them.
  Cursor next = at;
  int64_t load_x = place.begin + warp;
  if (load_x < place.end) next.step(a, rows, warp);
  const int step_row = 32 / chunks, step_col = 32 % chunks;  // from a lane's chunk to its next
  int page = -1;
  auto look_up = [&] {
    page = -1;
    if (load_x >= place.end) return;
    const int p = unit_slot(a, next.span, next.u) + (WHOLE ? 0 : lane);
    if (WHOLE || (lane < U && p >= next.span.lo && p < next.span.hi))
      page = c.table[(int64_t)next.b * c.max_pages + (p >> c.page_log2)];
  };
  look_up();
  auto load_unit = [&](int stage) {
    if (load_x < place.end) {
      const int p0 = unit_slot(a, next.span, next.u), kvh = next.r / a.tiles;
      const int p = p0 + lane;
      const bool in = lane < U && p >= next.span.lo && p < next.span.hi, ok = c.page_ok(page);
      if (in && !ok) report(kDevBadArgument);
      const uint32_t mask = __ballot_sync(0xffffffffu, in && ok);
      if (lane == 0) valid_of[warp][stage] = mask;
      const uint32_t dst = smem_u32(ring + stage * slot_bytes);
      // a row's number in the pool: below 2^32 (checked by tq4_paged_create)
      const uint32_t first = ((uint32_t)page * c.kv_heads + kvh) << c.page_log2;
      const int in_page = (1 << c.page_log2) - 1;
      if constexpr (WHOLE) {
        constexpr int C = DT / VN, PITCH = row_chunks<T>(DT) * 16;
        const int64_t off = (int64_t)(first + (p0 & in_page)) * (DT * (int)sizeof(T)) + lane * 16;
        const char* kp = static_cast<const char*>(a.k_pages) + off;
        const char* vp = static_cast<const char*>(a.v_pages) + off;
        const uint32_t to = dst + (lane / C) * PITCH + (lane % C) * 16;
        if (mask == (U == 32 ? 0xffffffffu : (1u << (U & 31)) - 1)) {
#pragma unroll
          for (int j = 0; j < U * C / 32; ++j) {
            const int at_row = j * 32 / C * PITCH + j * 32 % C * 16;
            cp_async16(to + at_row, kp + j * 512);
            cp_async16(to + U * PITCH + at_row, vp + j * 512);
          }
        } else {
#pragma unroll
          for (int j = 0; j < U * C / 32; ++j) {
            const int at_row = j * 32 / C * PITCH + j * 32 % C * 16;
            const bool take = (mask >> (lane / C + j * 32 / C)) & 1;
            cp_async16(to + at_row, take ? kp + j * 512 : a.k_pages, take);
            cp_async16(to + U * PITCH + at_row, take ? vp + j * 512 : a.v_pages, take);
          }
        }
      } else {
        const uint32_t row = first + (p & in_page);
        int i = lane / chunks, col = lane - i * chunks;
        for (int n = 0; n < U * chunks; n += 32) {  // every lane the same number of turns
          const int from = min(i, U - 1);
          const uint32_t rw = __shfl_sync(0xffffffffu, row, from);
          const bool take = (mask >> from) & 1;
          const int64_t off = take ? (int64_t)rw * (D * (int)sizeof(T)) + col * 16 : 0;
          if (i < U) {
            cp_async16(dst + i * row_bytes + col * 16, static_cast<const char*>(a.k_pages) + off, take);
            cp_async16(dst + (U + i) * row_bytes + col * 16, static_cast<const char*>(a.v_pages) + off, take);
          }
          i += step_row;
          col += step_col;
          if (col >= chunks) {
            col -= chunks;
            ++i;
          }
        }
      }
      load_x += kPartWarps;
      if (load_x < place.end) next.step(a, rows, kPartWarps);
      look_up();
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load_unit(s);

  Fold fold;
  int stage = 0;  // of the next unit to fold; the one before it is free
  for (int64_t x = place.begin; x < place.end;) {
    const int n = (int)min(place.end - x, (int64_t)(at.units - at.u));
    const int kvh = at.r / a.tiles, g0 = (at.r - kvh * a.tiles) * TILE;
    const int G = min(TILE, a.group - g0), h0 = kvh * a.group + g0;
    fold.begin(a, at.b, h0, G, qs, 0);
    // this warp's units of the row: those at a distance of warp, modulo kPartWarps, from the first
    const int mine = (int)((warp - (x - place.begin)) & (kPartWarps - 1));
    for (int i = mine; i < n; i += kPartWarps) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      load_unit(stage == 0 ? kStages - 1 : stage - 1);
      const int p0 = unit_slot(a, at.span, at.u + i);
      float* w = a.new_scores ? a.weights + (((int64_t)at.b * c.kv_heads + kvh) * c.max_slots + p0) * a.group + g0 : nullptr;
      fold.template fold<WHOLE>(a, ring + stage * slot_bytes, valid_of[warp][stage], row_bytes,
                                sizeof(T) == 2 ? (D + 15) / 16 : chunks, w, at.span.lo - p0, at.span.hi - p0, G, ps, qs);
      stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    // join the warps' parts; each leaves its o in the stage that it folded last
    const int free_stage = stage == 0 ? kStages - 1 : stage - 1;
    __syncwarp();
    fold.end(reinterpret_cast<float*>(ring + free_stage * slot_bytes), &ml[warp][0][0], D);
    if (lane == 0) free_of[warp] = free_stage;
    __syncthreads();
    const bool whole = n == at.units;
    const int64_t slot = (int64_t)blockIdx.x * 2 + (at.u > 0 ? 0 : 1);  // at most two rows of a CTA are not whole
    for (int i = tid; i < G * D; i += kPartThreads) {
      const int g = i / D;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kPartWarps; ++w) M = fmaxf(M, ml[w][g][0]);
      const float f = M == -INFINITY ? 0.f : M;
      float num = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < kPartWarps; ++w) {
        const float e = ex2(ml[w][g][0] - f);
        num = fmaf(e, reinterpret_cast<const float*>(dyn + (w * kStages + free_of[w]) * slot_bytes)[i], num);
        den = fmaf(e, ml[w][g][1], den);
      }
      if (whole) {
        static_cast<T*>(a.out)[((int64_t)at.b * a.heads + h0) * D + i] = from_f32<T>(den == 0.f ? 0.f : num / den);
        if (i == g * D) {
          a.stats[((int64_t)at.b * a.heads + h0 + g) * 2] = f;
          a.stats[((int64_t)at.b * a.heads + h0 + g) * 2 + 1] = den == 0.f ? 0.f : 1.f / den;
        }
      } else {
        a.parts[slot * TILE * D + i] = num;
        if (i == g * D) {
          a.ml[(slot * kMaxTile + g) * 2] = M;
          a.ml[(slot * kMaxTile + g) * 2 + 1] = den;
        }
      }
    }
    if (!whole && at.u > 0 && at.u + n == at.units) {
      info.end_b = at.b;
      info.end_r = at.r;
      info.first = cta_of(place.total, ctas, x - at.u);
    }
    __syncthreads();
    zero_tails(ring + free_stage * slot_bytes, 2 * U);
    x += n;
    if (x < place.end) at.step(a, rows, n);
  }
  if (tid == 0) a.info[blockIdx.x] = info;
}

// ---- the second kernel --------------------------------------------------------------------------
// Part slot of CTA k for a row that began in CTA `first`.
__device__ __forceinline__ int64_t part_slot(int k, int first) { return (int64_t)k * 2 + (k == first); }

// m (0 where nothing counts) and 1 / l of head g of a row that lies in CTAs first to last.
__device__ __forceinline__ float2 part_stats(const AttnArgs& a, int first, int last, int g) {
  float M = -INFINITY, den = 0.f;
  for (int k = first; k <= last; ++k) M = fmaxf(M, a.ml[(part_slot(k, first) * kMaxTile + g) * 2]);
  const float f = M == -INFINITY ? 0.f : M;
  for (int k = first; k <= last; ++k) {
    const float* p = a.ml + (part_slot(k, first) * kMaxTile + g) * 2;
    den = fmaf(ex2(p[0] - f), p[1], den);
  }
  return make_float2(f, den == 0.f ? 0.f : 1.f / den);
}

constexpr int kJoinThreads = 256;
constexpr int kJoinCols = 32;                         // 4-value columns of a block
constexpr int kJoinParts = kJoinThreads / kJoinCols;  // parts added at once
constexpr int kWeightBlocks = 4;                      // blocks that share a CTA's units

// blockIdx.x: a part CTA. blockIdx.y below join_blocks: some columns of the row that ends in it are
// joined; above: the weights of its units are added to the scores.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) attention_finish_kernel(const __grid_constant__ AttnArgs a, int join_blocks) {
  pdl_wait();
  pdl_trigger();
  __shared__ float4 sums[kJoinParts][kJoinCols];
  __shared__ float2 st[kMaxTile];
  const PagedView& c = a.cache;
  const int D = c.head_dim, tid = threadIdx.x;
  const PartInfo info = a.info[blockIdx.x];
  if ((int)blockIdx.y < join_blocks) {
    if (info.end_b < 0) return;
    const int kvh = info.end_r / a.tiles, g0 = (info.end_r - kvh * a.tiles) * a.tile;
    const int G = min(a.tile, a.group - g0), h0 = kvh * a.group + g0;
    const int first = info.first, last = blockIdx.x;
    const int col = blockIdx.y * kJoinCols + tid % kJoinCols, j = tid / kJoinCols;
    const int g = col * 4 / D;  // D is a multiple of 4
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    float2 ms = make_float2(0.f, 0.f);
    if (g < G) {
      ms = part_stats(a, first, last, g);
#pragma unroll 4
      for (int k = first + j; k <= last; k += kJoinParts) {
        const int64_t slot = part_slot(k, first);
        const float e = ex2(a.ml[(slot * kMaxTile + g) * 2] - ms.x);
        const float4 v = *reinterpret_cast<const float4*>(a.parts + slot * a.tile * D + col * 4);
        s.x = fmaf(e, v.x, s.x);
        s.y = fmaf(e, v.y, s.y);
        s.z = fmaf(e, v.z, s.z);
        s.w = fmaf(e, v.w, s.w);
      }
    }
    sums[j][tid % kJoinCols] = s;
    __syncthreads();
    if (j == 0 && g < G) {
      for (int i = 1; i < kJoinParts; ++i) {
        const float4 v = sums[i][tid];
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      T* out = static_cast<T*>(a.out) + ((int64_t)info.end_b * a.heads + h0) * D + col * 4;
      out[0] = from_f32<T>(s.x * ms.y);
      out[1] = from_f32<T>(s.y * ms.y);
      out[2] = from_f32<T>(s.z * ms.y);
      out[3] = from_f32<T>(s.w * ms.y);
    }
    return;
  }
  // scores: the rows of the heads' first tile, each with the heads of all tiles
  if (info.b < 0) return;
  const int ctas = active_ctas(a, info.total), rows = c.kv_heads * a.tiles;
  const int64_t end = first_unit(info.total, ctas, blockIdx.x + 1);
  int64_t x = first_unit(info.total, ctas, blockIdx.x), seq_first = info.seq_first;
  Cursor at;
  at.b = info.b;
  at.span = span_of(a, at.b);
  at.units = units_of(a, at.span);
  at.r = info.r;
  at.u = info.u0;
  const int part = blockIdx.y - join_blocks;
  while (x < end) {
    const int n = (int)min(end - x, (int64_t)(at.units - at.u));
    const int kvh = at.r / a.tiles;
    if (at.r == kvh * a.tiles) {
      const int64_t row = (int64_t)at.b * c.kv_heads + kvh;
      const float* old = a.scores + row * c.max_slots;
      float* now = a.new_scores + row * c.max_slots;
      // slots before the window keep theirs
      if (at.u == 0 && now != old)
        for (int p = part * kJoinThreads + tid; p < at.span.lo; p += kWeightBlocks * kJoinThreads) now[p] = old[p];
      const int p0 = max(at.span.lo, unit_slot(a, at.span, at.u)), p1 = min(at.span.hi, unit_slot(a, at.span, at.u + n));
      for (int t = 0; t < a.tiles; ++t) {
        const int g0 = t * a.tile, G = min(a.tile, a.group - g0);
        const int64_t x0 = seq_first + (int64_t)(at.r + t) * at.units;
        const int first = cta_of(info.total, ctas, x0), last = cta_of(info.total, ctas, x0 + at.units - 1);
        __syncthreads();
        if (tid < G) {
          const float* s = a.stats + ((int64_t)at.b * a.heads + kvh * a.group + g0 + tid) * 2;
          st[tid] = first == last ? make_float2(s[0], s[1]) : part_stats(a, first, last, tid);
        }
        __syncthreads();
        for (int p = p0 + part * kJoinThreads + tid; p < p1; p += kWeightBlocks * kJoinThreads) {
          const float* w = a.weights + (row * c.max_slots + p) * a.group + g0;
          float sum = 0.f;
          for (int g = 0; g < G; ++g) sum = fmaf(ex2(w[g] - st[g].x), st[g].y, sum);
          now[p] = (t == 0 ? old[p] : now[p]) + sum;
        }
      }
    }
    x += n;
    if (x < end) {
      if (at.r + 1 == rows) seq_first += (int64_t)rows * at.units;
      at.step(a, rows, n);
    }
  }
}

namespace {

int head_tile(const tq4_paged_desc& d, int heads) {
  const int group = heads / d.kv_heads;
  if (d.dtype == TQ4_F32) return group >= 5 ? 8 : group >= 3 ? 4 : group;
  return group > 8 ? 16 : 8;
}

// Offsets of the workspace's parts, in bytes, each a multiple of 16.
struct Workspace {
  int64_t stats, ml, parts, weights, bytes;
};
Workspace workspace_of(const tq4_paged_desc& d, int heads, int64_t batch, bool with_scores) {
  auto up = [](int64_t n) { return (n + 15) / 16 * 16; };
  Workspace w;
  w.stats = up(kMaxCtas * sizeof(PartInfo));
  w.ml = w.stats + up(batch * heads * 2 * 4);
  w.parts = w.ml + kMaxCtas * 2 * kMaxTile * 2 * 4;
  w.weights = w.parts + up((int64_t)kMaxCtas * 2 * head_tile(d, heads) * d.head_dim * 4);
  w.bytes = w.weights + (with_scores ? up(batch * heads * (int64_t)d.max_pages * d.page_size * 4) : 0);
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

template <typename T, int DT, int TILE>
tq4_status launch_part(AttnArgs& a, cudaStream_t st) {
  a.unit = FoldOf<T, DT, TILE>::U;
  while ((1 << a.unit_log2) < a.unit) ++a.unit_log2;
  a.ctas = DT <= 128 ? kMaxCtas : kSms;
  const bool whole = a.cache.head_dim == DT && (1 << a.cache.page_log2) >= a.unit;
  const auto kern = whole ? attention_part_kernel<T, DT, TILE, true> : attention_part_kernel<T, DT, TILE, false>;
  static std::atomic<uint64_t> set[2];  // per device, per instantiation
  TQ4_CUDA(set_smem_limit_once(kern, part_smem<T, DT, TILE>(DT), set[whole]));
  TQ4_CUDA(launch_pdl(kern, dim3(a.ctas), dim3(kPartThreads), part_smem<T, DT, TILE>(a.cache.head_dim), st, a));
  return TQ4_OK;
}

template <typename T, int TILE>
tq4_status launch_width(AttnArgs& a, cudaStream_t st) {
  const int D = a.cache.head_dim;
  if (D <= 64) return launch_part<T, 64, TILE>(a, st);
  if (D <= 128) return launch_part<T, 128, TILE>(a, st);
  return launch_part<T, 256, TILE>(a, st);
}

template <typename T>
tq4_status launch_attention(AttnArgs& a, cudaStream_t st) {
  if constexpr (sizeof(T) == 4) {
    switch (a.tile) {
      case 1: TQ4_TRY((launch_width<T, 1>(a, st))); break;
      case 2: TQ4_TRY((launch_width<T, 2>(a, st))); break;
      case 4: TQ4_TRY((launch_width<T, 4>(a, st))); break;
      default: TQ4_TRY((launch_width<T, 8>(a, st))); break;
    }
  } else {
    if (a.tile == 8) TQ4_TRY((launch_width<T, 8>(a, st)));
    else TQ4_TRY((launch_width<T, 16>(a, st)));
  }
  const int join = (std::min(a.tile, a.group) * a.cache.head_dim / 4 + kJoinCols - 1) / kJoinCols;
  TQ4_CUDA(launch_pdl(attention_finish_kernel<T>, dim3(a.ctas, join + (a.new_scores ? kWeightBlocks : 0)),
                      dim3(kJoinThreads), 0, st, a, join));
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
  *bytes = workspace_of(cache->desc, heads, batch, with_scores != 0).bytes;
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
  if (workspace_bytes < ws.bytes || !aligned16(workspace)) {
    set_error("tq4_paged_attention: the workspace must be 16-byte aligned and hold %lld bytes, got %lld",
              (long long)ws.bytes, (long long)workspace_bytes);
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
  a.tile = head_tile(d, heads);
  a.tiles = (a.group + a.tile - 1) / a.tile;
  a.q_even = (reinterpret_cast<uintptr_t>(q) & 3) == 0 && (q_stride & 1) == 0;
  a.scale2 = scale * kLog2e;
  a.scores = scores;
  a.new_scores = new_scores;
  char* w = static_cast<char*>(workspace);
  a.info = reinterpret_cast<PartInfo*>(w);
  a.stats = reinterpret_cast<float*>(w + ws.stats);
  a.ml = reinterpret_cast<float*>(w + ws.ml);
  a.parts = reinterpret_cast<float*>(w + ws.parts);
  a.weights = reinterpret_cast<float*>(w + ws.weights);
  DeviceGuard guard(cache->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (d.dtype) {
    case TQ4_F16: return launch_attention<__half>(a, st);
    case TQ4_BF16: return launch_attention<__nv_bfloat16>(a, st);
    default: return launch_attention<float>(a, st);
  }
}

}  // extern "C"
