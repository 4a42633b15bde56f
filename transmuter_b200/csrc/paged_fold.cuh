// What the paged attention's kernels share with their folds (paged_attention.cu): the arguments, and the two ways
// to fold a unit of keys and values, already in shared memory, into a row's running softmax.
#pragma once

#include "paged.cuh"
#include "sm100.cuh"

namespace tq4 {

constexpr int kStages = 3;
constexpr int kSms = 148;  // of a B200; only a grid's size, no CTA waits for another
constexpr int kLevels = 6;
// A chunk has three units of each of four warps at least where there are chunks to take: a warp's loads and
// page lookups run three units ahead, so they need no more than the chunk after the current one.
constexpr int kMinChunk = 12;
constexpr int kMaxTile = 16;  // query heads of a row at most
constexpr float kLog2e = 1.4426950408889634f;

// How the line is cut: into `ctas` shares of `share` units, the first `extra` of them one longer, and each share
// into `levels` chunks, which begin at base[level] of it. (Every share holds chunks of all sizes, so that no
// row is made of small ones alone.)
struct Plan {
  int64_t total;  // units
  int64_t share;
  int64_t base[kLevels];
  int32_t ctas, levels, extra;
};

struct __align__(16) Chunk {
  int32_t b, r, u, n;  // sequence, row of it, unit of the row that the chunk begins with; units. b < 0: none
  int32_t units;       // of that row
  int32_t index;       // the chunk's number along the line
  int64_t seq_first;   // the line's place where sequence b begins
};
__device__ __forceinline__ Chunk no_chunk() { return {-1, 0, 0, 0, 0, 0, 0}; }

struct AttnArgs {
  PagedView cache;
  const void *q, *k_pages, *v_pages;
  int64_t q_stride;
  void* out;
  const int32_t* lengths;
  int64_t batch, window;
  int heads, group;  // query heads, those of a KV head
  int tile, tiles;   // heads of a row, and rows of a KV head
  int unit, unit_log2;  // slots of a unit
  int warps, ctas, levels;  // of a CTA; CTAs the line is cut for; sizes of chunks at most
  int cluster;              // CTAs of a row where there is no line, else 0
  int q_even;        // q's heads are 4-byte aligned
  float scale2;      // scale * log2(e): scores are kept for exp2
  const float* scores;
  float* new_scores;
  // workspace
  Plan* plan;
  int64_t* seq_first;  // [batch]: the line's place where a sequence begins; written and read where there are scores
  uint8_t* ends;       // [grid * warps], by piece: 1 where a row ends that began in an earlier one
  int4* joins;         // [grid * warps]: that row: sequence, row, the piece it began in
  float* stats;    // [batch][heads][2]: m, 1 / l of rows that lie in one piece
  // The parts of other rows: a piece has two at most, of a row that began in an earlier one (0) and of one that
  // ends in a later one (1). A row's parts of a head lie in a run, so that the join streams them (with a
  // piece's heads in a run instead, the strides met few memory channels: 26 us for 8 rows of 592 parts).
  int pieces;      // grid * warps
  float* ml;       // [2][tile][pieces][2]: m, l
  float* parts;    // [2][tile][pieces][head_dim]: o
  float* weights;  // [batch][kv_heads][max_slots][group]: scores times scale2
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
// 2^15 (kScale) as they are rounded, so that weights down to 2^-29 of the largest keep f16's full precision; o carries
// that factor until the row's end. (Taken off m instead, the 15 was itself rounded where scores are 2^24 and more, to
// 16 from 2^26 on, and the largest weight came to 2^16, which f16 does not hold.)
template <typename T, int DT, int TILE>
struct MmaFold {
  static constexpr int U = DT == 64 ? 32 : 16;
  static constexpr int NT = TILE / 8;  // column blocks of heads
  static constexpr int KS = DT / 16;   // 16-value steps of a row
  static constexpr float kScale = std::is_same_v<T, __half> ? 32768.f : 1.f;
  uint32_t qf[NT][KS][2];
  float o[NT][KS][4];
  float m[NT][2], l[NT][2];  // heads 2 * (lane % 4) + {0, 1} of each block

  __device__ __forceinline__ void load_q(const AttnArgs& a, int64_t b, int h0, int G, float*) {
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
    }
  }
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
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
        }
      if (w)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int slot = t * 16 + (lane >> 2) + h * 8, g = n * 8 + (lane & 3) * 2;
            if (slot < from || slot >= to || g >= G) continue;
            float* p = w + slot * a.group + g;
            if ((a.group & 1) == 0) {
              *reinterpret_cast<float2*>(p) = make_float2(s[t][n][2 * h], s[t][n][2 * h + 1]);
            } else {
              p[0] = s[t][n][2 * h];
              if (g + 1 < G) p[1] = s[t][n][2 * h + 1];
            }
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
        mx[j] = fmaxf(m[n][j], mx[j]);
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
        pf[t][n][0] = transpose8x8(pack2<T>(p[0] * kScale, p[1] * kScale));
        pf[t][n][1] = transpose8x8(pack2<T>(p[2] * kScale, p[3] * kScale));
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

  // The row's end: of G heads, o / l to out[G][D] and m, 1 / l to ml[G][2], or where the row is not whole (out is
  // null) o to part[G][pieces][D] and m, l to ml[G][pieces][2].
  __device__ __forceinline__ void end(T* out, float* part, float* ml, int64_t pieces, int G, int D) {
    const int lane = threadIdx.x & 31;
    constexpr float kOnce = 1.f / kScale;  // a power of two: exact
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        for (int off = 4; off < 32; off <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], off);
        const int g = n * 8 + (lane & 3) * 2 + j;
        if (g >= G) continue;
        const float inv = l[n][j] == 0.f ? 0.f : 1.f / l[n][j];
        if (lane < 4)
          *reinterpret_cast<float2*>(ml + 2 * (out ? g : g * pieces)) =
              out ? make_float2(m[n][j] == -INFINITY ? 0.f : m[n][j], inv) : make_float2(m[n][j], l[n][j]);
        float* to = part + g * pieces * D;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const int d = k * 16 + (lane >> 2);
          if (out) {
            if (d < D) out[g * D + d] = from_f32<T>(o[n][k][j] * (inv * kOnce));
            if (d + 8 < D) out[g * D + d + 8] = from_f32<T>(o[n][k][j + 2] * (inv * kOnce));
          } else {
            if (d < D) to[d] = o[n][k][j] * kOnce;
            if (d + 8 < D) to[d + 8] = o[n][k][j + 2] * kOnce;
          }
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
  static constexpr int HALVES = DT == 64 ? 2 : 1;  // rows of up to 16 chunks: each half of the warp has every other slot
  static constexpr int N = 4 * TILE;
  static constexpr int STEPS = PG == 2 ? 4 : 3;
  static constexpr int LEFT = (N >> STEPS) > 0 ? (N >> STEPS) : 1;             // sums a lane ends with
  static constexpr int COPIES = (1 << STEPS) > N ? (1 << STEPS) / N : 1;       // lanes that end with the same
  float o[COLS][4][TILE];
  float m, l;  // of the head that this lane's sums belong to
  int idx;     // they are numbers idx, idx + 1, ...: head idx / 4, slots idx % 4

  // q to the warp's qs[TILE][D]
  __device__ __forceinline__ void load_q(const AttnArgs& a, int64_t b, int h0, int G, float* qs) {
    const int D = a.cache.head_dim;
    const float* src = static_cast<const float*>(a.q) + b * a.q_stride + (int64_t)h0 * D;
    __syncwarp();
    for (int i = threadIdx.x & 31; i < TILE * D; i += 32) qs[i] = i < G * D ? src[i] : 0.f;
    __syncwarp();
  }
  __device__ __forceinline__ void begin() {
    const int lane = threadIdx.x & 31;
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
    for (int i = 0; i < U / HALVES; ++i) {
      const int slot = HALVES == 1 ? i : 2 * i + (lane >> 4), chunk = HALVES == 1 ? lane : lane & 15;
      alignas(16) float p[TILE];
      if constexpr (TILE >= 4) {
#pragma unroll
        for (int g = 0; g < TILE; g += 4)
          *reinterpret_cast<float4*>(p + g) = *reinterpret_cast<const float4*>(ps + slot * TILE + g);
      } else {
#pragma unroll
        for (int g = 0; g < TILE; ++g) p[g] = ps[slot * TILE + g];
      }
#pragma unroll
      for (int j = 0; j < COLS; ++j)
        if (chunk + j * 32 < chunks) {
          const float4 x = *reinterpret_cast<const float4*>(vs + slot * row_bytes + (chunk + j * 32) * 16);
#pragma unroll
          for (int g = 0; g < TILE; ++g) {
            o[j][0][g] = fmaf(p[g], x.x, o[j][0][g]);
            o[j][1][g] = fmaf(p[g], x.y, o[j][1][g]);
            o[j][2][g] = fmaf(p[g], x.z, o[j][2][g]);
            o[j][3][g] = fmaf(p[g], x.w, o[j][3][g]);
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

  __device__ __forceinline__ void end(float* out, float* part, float* ml, int64_t pieces, int G, int D) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int off = 16 / TILE; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    l *= 1.f / COPIES;
    if constexpr (HALVES == 2)
#pragma unroll
      for (int g = 0; g < TILE; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][e][g] += __shfl_xor_sync(0xffffffffu, o[0][e][g], 16);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if ((lane & (32 / TILE - 1)) == 0 && (idx >> 2) < G)
      *reinterpret_cast<float2*>(ml + 2 * (idx >> 2) * (out ? 1 : pieces)) =
          out ? make_float2(m == -INFINITY ? 0.f : m, inv) : make_float2(m, l);
#pragma unroll
    for (int g = 0; g < TILE; ++g) {
      const float f = out ? __shfl_sync(0xffffffffu, inv, g * (32 / TILE)) : 1.f;
#pragma unroll
      for (int j = 0; j < COLS; ++j)
        if (g < G && (lane + j * 32) * 4 < D) {  // (with HALVES the first half has all columns)
          float* p = (out ? out + g * D : part + g * pieces * D) + (lane + j * 32) * 4;  // out may be aligned to 4 bytes only
          p[0] = o[j][0][g] * f;
          p[1] = o[j][1][g] * f;
          p[2] = o[j][2][g] * f;
          p[3] = o[j][3][g] * f;
        }
    }
  }
};

template <typename T, int DT, int TILE>
using FoldOf = std::conditional_t<sizeof(T) == 4, FmaFold<DT, TILE>, MmaFold<T, DT, TILE>>;

}  // namespace tq4
