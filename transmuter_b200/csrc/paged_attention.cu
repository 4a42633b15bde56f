// Attention of one new token of each sequence over the paged cache (include/tq4_paged.h).
//
// A cache row is read once and used by the query heads of its KV head alone, so memory bounds this:
// 2 * head_dim values a slot and KV head. The kernels are built around keeping loads in flight.
//
// The work is split over the cache's length without the host knowing any length. A sequence's slots are
// cut into units of U (8 to 32, a warp's step), and all units of all (sequence, KV head, head tile)
// rows stand in one line. It is cut into a share for each of the P CTAs that run at once, and each share into
// chunks: five eighths of it, then of what is left, and so on (at most kLevels, kMinChunk units at least).
// A CTA of the grid is a chunk; one that has begun its chunk asks the hardware for the next that has not
// begun (cluster launch control) and goes on with it, so that its loads never pause. SMs get unequal
// shares of the memory's rate (with one equal part for each CTA, the first was done at 125 us and the
// last at 183 us of 64 sequences of 4096 slots): the small chunks at the end even that out.
//   part    A CTA finds its chunk by a prefix sum over the lengths. Its warps take runs of the chunk's units
//           (pieces, one for each warp, whoever is free) without waiting for one another: each has a ring of
//           kStages units of its own that cp.async fills, also across the borders of rows and pieces. A warp folds
//           units into a running maximum m, a sum l of exp2(s - m) and an unnormalised output o (online
//           softmax). A row inside one piece is finished there; of others the parts go to the workspace.
//           (With the warps of a CTA joined in shared memory at each row's end, that end took 2.2 us, and
//           four of them a sixth of the kernel's time for 32 sequences of up to 4096 slots.)
//   finish  joins the parts in the line's order, so that results depend on the call's sizes and lengths alone and
//           not on who took which chunk, and adds the softmax weights to the scores.
#include "paged_fold.cuh"

namespace tq4 {

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

// a / b of values that hardly ever pass 32 bits, where a division takes a fifth of the time.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}
// First unit of the chunk that is number c along the line.
__device__ __forceinline__ int64_t chunk_first(const Plan& p, int c) {
  const int i = c / p.levels, level = c - i * p.levels;
  return i * p.share + min(i, p.extra) + (i < p.ctas ? p.base[level] : 0);
}
// The chunk that holds unit x.
__device__ __forceinline__ int chunk_of(const Plan& p, int64_t x) {
  const int64_t longer = p.extra * (p.share + 1);
  const int i = x < longer ? (int)divide(x, p.share + 1) : p.extra + (int)divide(x - longer, p.share);
  const int64_t off = x - (i * p.share + min(i, p.extra));
  int level = 0;
  while (level + 1 < p.levels && off >= p.base[level + 1]) ++level;
  return i * p.levels + level;
}

// A chunk of n units is cut into a piece for each warp.
__device__ __forceinline__ int piece_first(int n, int warps, int warp) { return (int)((int64_t)n * warp / warps); }
// The piece that holds unit x, counted over all chunks.
__device__ __forceinline__ int piece_of(const Plan& p, int warps, int64_t x) {
  const int c = chunk_of(p, x);
  const int64_t first = chunk_first(p, c);
  return c * warps + (int)divide((x - first + 1) * warps - 1, chunk_first(p, c + 1) - first);
}

// The line as a CTA of THREADS threads sees it: each thread sums a run of sequences.
template <int THREADS> struct Line {
  Plan plan;
  int64_t ends[THREADS];  // where each run ends
  int per;                // sequences of a run
};
// Every thread of the block calls it; ends with a barrier.
template <int THREADS>
__device__ __forceinline__ void make_line(const AttnArgs& a, Line<THREADS>& line, int64_t* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t rows = (int64_t)a.cache.kv_heads * a.tiles;
  const int per = (int)((a.batch + THREADS - 1) / THREADS);
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
  int64_t before = 0, total = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w == warp) before = total;
    total += red[w];
  }
  line.ends[tid] = before + incl;
  if (tid == 0) {
    Plan& p = line.plan;
    line.per = per;
    p.total = total;
    // a short line is not spread thin: each warp gets a unit at least
    p.ctas = (int)min((int64_t)a.ctas, divide(total + a.warps - 1, a.warps));
    p.levels = 0;
    if (total > 0) {
      p.share = divide(total, p.ctas);
      p.extra = (int32_t)(total - p.share * p.ctas);
      p.base[0] = 0;
      p.levels = 1;
      for (int64_t left = p.share; p.levels < a.levels && left >= 2 * kMinChunk; ++p.levels) {
        left = max(left * 3 / 8, (int64_t)kMinChunk);
        p.base[p.levels] = p.share - left;
      }
    }
  }
  __syncthreads();
}

// Chunk `number` of those that the grid's CTAs are, the first of all shares and then the second, by a warp.
template <int THREADS>
__device__ __forceinline__ Chunk find_chunk(const AttnArgs& a, const Line<THREADS>& line, int number) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)a.cache.kv_heads * a.tiles;
  const int level = number / line.plan.ctas, c = (number - level * line.plan.ctas) * line.plan.levels + level;
  const int64_t x = chunk_first(line.plan, c);
  int below = 0;  // runs that end at or before x
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) below += __popc(__ballot_sync(0xffffffffu, line.ends[i * 32 + lane] <= x));
  Chunk k;
  k.seq_first = below ? line.ends[below - 1] : 0;
  for (k.b = line.per * below;; ++k.b) {
    k.units = units_of(a, span_of(a, k.b));
    if (x < k.seq_first + k.units * rows) break;
    k.seq_first += k.units * rows;
  }
  k.r = (int)divide(x - k.seq_first, k.units);
  k.u = (int)((x - k.seq_first) - (int64_t)k.r * k.units);
  k.n = (int)(chunk_first(line.plan, c + 1) - x);
  k.index = c;
  return k;
}

// Cluster launch control: asks for a CTA of this grid that has not begun, which then never does; the
// answer (16 bytes) arrives at `to`, completing on `bar`.
__device__ __forceinline__ void ask_for_cta(uint32_t to, uint32_t bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(to), "r"(bar)
               : "memory");
}
// The CTA's number, or -1 where all have begun (then there is no use in asking again, and no leave).
__device__ __forceinline__ int asked_cta(uint32_t from) {
  uint32_t got, x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(from)
      : "memory");
  return got ? (int)x : -1;
}

// A place in the line, stepped forward.
struct Cursor {
  int b, r, u, units;
  Span span;
  __device__ __forceinline__ void set(const AttnArgs& a, const Chunk& c) {
    b = c.b;
    r = c.r;
    u = c.u;
    span = span_of(a, b);
    units = units_of(a, span);
  }
  // `n` units on; the caller knows that the chunk goes that far.
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

// Warps of a CTA: four, or three where f32 queries of 8 heads need their room.
template <typename T, int TILE> constexpr int kWarpsOf = sizeof(T) == 4 && TILE == 8 ? 3 : 4;

// Dynamic shared memory: the rings, then for f32 each warp's queries and softmax weights.
template <typename T, int DT, int TILE> constexpr int part_smem(int head_dim) {
  constexpr int U = FoldOf<T, DT, TILE>::U;
  return kWarpsOf<T, TILE> * (kStages * 2 * U * row_chunks<T>(head_dim) * 16 +
                              (sizeof(T) == 4 ? TILE * head_dim * 4 + U * TILE * 4 : 0));
}

// Sends for a unit of KV head kvh, its keys and behind them its values, from slot p0 on. `page` is where lane i's
// slot lies (look_up_page). *valid gets a bit for each slot that counts; rows of others may hold anything, NaN too, and become
// zeros.
//
// WHOLE: head_dim is DT, so that a lane's chunks lie in rows and columns known to the compiler. Where a page holds
// whole units too, a unit's keys are one run of memory, as are its values, and all offsets are constants (the loads
// of a unit then take 30 instructions a lane instead of 300).
template <typename T, int DT, int U, bool WHOLE>
__device__ __forceinline__ void load_rows(const AttnArgs& a, char* slot, uint32_t* valid, Span span, int p0, int kvh, int page) {
  constexpr int VN = 16 / sizeof(T);
  const PagedView& c = a.cache;
  const int lane = threadIdx.x & 31, D = WHOLE ? DT : c.head_dim, chunks = D / VN, row_bytes = row_chunks<T>(D) * 16;
  const int p = p0 + lane;
  const bool in = lane < U && p >= span.lo && p < span.hi, ok = c.page_ok(page);
  if (in && !ok) report(kDevBadArgument);
  const uint32_t mask = __ballot_sync(0xffffffffu, in && ok);
  if (lane == 0) *valid = mask;
  const uint32_t dst = smem_u32(slot);
  // a row's number in the pool: below 2^32 (checked by tq4_paged_create)
  const uint32_t first = ((uint32_t)page * c.kv_heads + kvh) << c.page_log2;
  const int in_page = (1 << c.page_log2) - 1;
  if constexpr (WHOLE) {
    constexpr int C = DT / VN, PITCH = row_chunks<T>(DT) * 16;
    const uint32_t to = dst + (lane / C) * PITCH + (lane % C) * 16;
    if ((1 << c.page_log2) < U) {  // smaller pages: a lane's rows by shuffle
      const uint32_t row = first + (p & in_page);
#pragma unroll
      for (int j = 0; j < U * C / 32; ++j) {
        const int at_row = j * 32 / C * PITCH + j * 32 % C * 16, from = lane / C + j * 32 / C;
        const uint32_t rw = __shfl_sync(0xffffffffu, row, from);
        const bool take = (mask >> from) & 1;
        const int64_t off = take ? (int64_t)rw * (DT * (int)sizeof(T)) + (lane % C) * 16 + j * 32 % C * 16 : 0;
        cp_async16(to + at_row, static_cast<const char*>(a.k_pages) + off, take);
        cp_async16(to + U * PITCH + at_row, static_cast<const char*>(a.v_pages) + off, take);
      }
      return;
    }
    const int64_t off = (int64_t)(first + (p0 & in_page)) * (DT * (int)sizeof(T)) + lane * 16;
    const char* kp = static_cast<const char*>(a.k_pages) + off;
    const char* vp = static_cast<const char*>(a.v_pages) + off;
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
    const int step_row = 32 / chunks, step_col = 32 % chunks;  // from a lane's chunk to its next
    int i = lane / chunks, col = lane - i * chunks;
    if ((1 << c.page_log2) >= U) {  // the unit is one run of memory here too
      const uint32_t row0 = __shfl_sync(0xffffffffu, first, mask ? __ffs(mask) - 1 : 0) + (p0 & in_page);
      const int64_t off = (int64_t)row0 * (D * (int)sizeof(T)) + lane * 16;
      const char* kp = static_cast<const char*>(a.k_pages) + off;
      const char* vp = static_cast<const char*>(a.v_pages) + off;
      uint32_t to = dst + i * row_bytes + col * 16;
      const int step = step_row * row_bytes + step_col * 16, wrap = row_bytes - chunks * 16;
      for (int n = lane; n < U * chunks; n += 32) {
        const bool take = (mask >> i) & 1;
        cp_async16(to, take ? kp : a.k_pages, take);
        cp_async16(to + U * row_bytes, take ? vp : a.v_pages, take);
        kp += 512;
        vp += 512;
        to += step;
        i += step_row;
        col += step_col;
        if (col >= chunks) {
          col -= chunks;
          to += wrap;
          ++i;
        }
      }
      return;
    }
    const uint32_t row = first + (p & in_page);
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
}
// The page of the unit's slot p0 + lane, -1 outside the span; where a page holds whole units and rows are WHOLE
// (load_rows), the unit's page in every lane.
template <int U, bool WHOLE>
__device__ __forceinline__ int look_up_page(const AttnArgs& a, int b, Span span, int p0) {
  const bool one = WHOLE && (1 << a.cache.page_log2) >= U;
  const int lane = threadIdx.x & 31, p = one ? p0 : p0 + lane;
  if (one || (lane < U && p >= span.lo && p < span.hi))
    return a.cache.table[(int64_t)b * a.cache.max_pages + (p >> a.cache.page_log2)];
  return -1;
}
// 16-bit rows of an odd number of 16-byte chunks: their last 16-value step reads one more, kept at zero.
template <typename T>
__device__ __forceinline__ void zero_tails(char* ring, int n_rows, int head_dim) {
  const int chunks = head_dim * (int)sizeof(T) / 16;
  if (sizeof(T) == 2 && (chunks & 1))
    for (int i = threadIdx.x & 31; i < n_rows; i += 32)
      *reinterpret_cast<uint4*>(ring + i * row_chunks<T>(head_dim) * 16 + chunks * 16) = make_uint4(0, 0, 0, 0);
}

// ---- part -----------------------------------------------------------------------------------------
template <typename T, int DT, int TILE, bool WHOLE>
__global__ void __launch_bounds__(kWarpsOf<T, TILE> * 32, DT <= 128 ? 2 : 1)
    attention_part_kernel(const __grid_constant__ AttnArgs a) {
  using Fold = FoldOf<T, DT, TILE>;
  constexpr int U = Fold::U, WARPS = kWarpsOf<T, TILE>, THREADS = WARPS * 32;
  constexpr int VN = 16 / sizeof(T);
  __shared__ uint32_t valid_of[WARPS][kStages];
  __shared__ Line<THREADS> line;
  __shared__ int64_t red[WARPS];
  __shared__ Chunk chunk_at[4];  // the CTA's chunks after the first, by turns
  __shared__ __align__(16) uint4 answer;
  __shared__ __align__(8) uint64_t known[4];  // chunk_at[i] holds a chunk
  __shared__ __align__(8) uint64_t taken[4];  // all its pieces have been taken
  __shared__ __align__(8) uint64_t answered;
  __shared__ int s_abort, s_taken, s_ask, s_answers;
  extern __shared__ __align__(16) char dyn[];
  const PagedView& c = a.cache;
  const int D = WHOLE ? DT : c.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int chunks = D / VN, row_bytes = row_chunks<T>(D) * 16;
  const int slot_bytes = 2 * U * row_bytes;
  char* ring = dyn + warp * kStages * slot_bytes;
  float* qs = reinterpret_cast<float*>(dyn + WARPS * kStages * slot_bytes) + warp * TILE * (D + U);
  float* ps = qs + TILE * D;
  const int rows = c.kv_heads * a.tiles;

  zero_tails<T>(ring, kStages * 2 * U, D);
  if (tid == 0) {
    s_abort = 0;
    s_taken = WARPS;  // each warp has a piece of the first chunk
    s_ask = (int)gridDim.x > a.ctas;
    s_answers = 0;
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&known[i]), 1);
      mbar_init(smem_u32(&taken[i]), WARPS);
    }
    mbar_init(smem_u32(&answered), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  make_line(a, line, red);
  const int n_chunks = line.plan.ctas * line.plan.levels;
  // The second kernel needs the plan, and for the scores where each sequence begins. Every CTA that begins and has a
  // chunk writes them, all the same values: any one of them, the first too, may be taken by another before it begins,
  // but whoever takes one has begun and has a chunk itself. (Where there is no chunk, none is taken.)
  if ((int)blockIdx.x < n_chunks || blockIdx.x == 0) {
    if (tid == 0) *a.plan = line.plan;
    if (a.new_scores) {
      int64_t at = tid ? line.ends[tid - 1] : 0;
      for (int b = tid * line.per; b < (tid + 1) * line.per && b < a.batch; ++b) {
        a.seq_first[b] = at;
        at += (int64_t)units_of(a, span_of(a, b)) * rows;
      }
    }
  }
  if ((int)blockIdx.x >= n_chunks) return;  // the grid was made for longer sequences

  // ---- the CTA's pieces ----
  // Piece j is one of chunk j / WARPS of the CTA (0 is blockIdx.x). Warps take them by ticket; who takes the
  // first of a chunk makes it known to the others and asks for the one after it. That happens in the chunks'
  // order: a warp waits with one piece at most. Numbers beyond the line's chunks are asked for too, so that
  // they need not be launched.
  const bool seamless = line.plan.levels > 1;  // loads go on into the next piece; a single level's may be too short
  auto draw = [&] {
    if (lane == 0 && s_ask) ask_for_cta(smem_u32(&answer), smem_u32(&answered));
    __syncwarp();
  };
  auto drawn = [&]() -> Chunk {
    while (s_ask) {
      const int n = s_answers;
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&answered), n & 1, &s_abort, kDevTimeoutAttn))) break;
      const int got = asked_cta(smem_u32(&answer));
      fence_proxy_async_smem();  // the answer is read before the next one is written
      __syncwarp();
      if (lane == 0) {
        s_answers = n + 1;
        if (got < 0) s_ask = 0;
      }
      __syncwarp();
      if (got >= n_chunks) draw();
      else if (got >= 0) return find_chunk(a, line, got);
    }
    return no_chunk();
  };
  struct Piece {
    Chunk k;
    int w;  // which of the chunk's
  };
  auto take = [&]() -> Piece {
    int j = 0;
    if (lane == 0) j = atomicAdd(&s_taken, 1);
    j = __shfl_sync(0xffffffffu, j, 0);
    const int s = j / WARPS, at = s & 3, phase = (s - 1) >> 2;
    Piece p = {no_chunk(), j - s * WARPS};
    if (p.w == 0) {
      const Chunk k = drawn();
      if (s > 4 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&taken[at]), (phase - 1) & 1, &s_abort, kDevTimeoutAttn))) return p;
      if (lane == 0) {
        chunk_at[at] = k;
        mbar_arrive(smem_u32(&known[at]));
      }
      __syncwarp();
      if (k.b >= 0) draw();
    }
    if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&known[at]), phase & 1, &s_abort, kDevTimeoutAttn))) return p;
    p.k = chunk_at[at];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&taken[at]));
    return p;
  };

  // ---- this warp's loads ----
  // A unit's pages are looked up one unit ahead of their use.
  Piece cur = {find_chunk(a, line, blockIdx.x), warp};  // being folded
  Piece coming = cur;                                   // being loaded
  if (warp == 0) draw();
  Cursor next;
  int load_left;
  auto enter = [&] {  // sets the loads to `coming`
    load_left = 0;
    if (coming.k.b < 0) return;
    const int first = piece_first(coming.k.n, WARPS, coming.w);
    load_left = piece_first(coming.k.n, WARPS, coming.w + 1) - first;
    if (load_left == 0) return;
    next.set(a, coming.k);
    if (first) next.step(a, rows, first);
  };
  auto advance = [&] {
    if (--load_left > 0) {
      next.step(a, rows, 1);
    } else if (seamless) {
      coming = take();
      enter();
    }
  };
  auto look_up = [&]() -> int {
    return load_left ? look_up_page<U, WHOLE>(a, next.b, next.span, unit_slot(a, next.span, next.u)) : -1;
  };
  auto load_unit = [&](int stage, const Cursor& at, int page) {
    load_rows<T, DT, U, WHOLE>(a, ring + stage * slot_bytes, &valid_of[warp][stage], at.span,
                               unit_slot(a, at.span, at.u), at.r / a.tiles, page);
  };

  // ---- folding ----
  Fold fold;
  int stage = 0;  // of the next unit to fold; the one before it is free
  enter();
  int page = -1;
  auto start = [&] {  // the first two units' pages are looked up together
    static_assert(kStages == 3);
    const Cursor c0 = next;
    const bool any = load_left > 0;
    const int page0 = look_up();
    if (any) advance();
    const int page1 = look_up();
    if (any) load_unit(stage, c0, page0);
    cp_async_commit();
    if (load_left > 0) {
      load_unit(stage == kStages - 1 ? 0 : stage + 1, next, page1);
      advance();
    }
    cp_async_commit();
    page = look_up();
  };
  start();
  for (;;) {
    const int piece = cur.k.index * WARPS + cur.w;
    const int first = piece_first(cur.k.n, WARPS, cur.w);
    int left = piece_first(cur.k.n, WARPS, cur.w + 1) - first;
    bool ends = false;
    if (left == 0)  // parts that the second kernel passes over
      for (int i = lane; i < 2 * TILE; i += 32)
        *reinterpret_cast<float2*>(a.ml + ((int64_t)i * a.pieces + piece) * 2) = make_float2(-INFINITY, 0.f);
    Cursor at;
    if (left > 0) {
      at.set(a, cur.k);
      if (first) at.step(a, rows, first);
    }
    while (left > 0) {
      const int n = min(left, at.units - at.u);
      const int kvh = at.r / a.tiles, g0 = (at.r - kvh * a.tiles) * TILE;
      const int G = min(TILE, a.group - g0), h0 = kvh * a.group + g0;
      fold.load_q(a, at.b, h0, G, qs);
      fold.begin();
      for (int i = 0; i < n; ++i) {
        cp_async_wait<kStages - 2>();
        __syncwarp();
        if (load_left > 0) {
          load_unit(stage == 0 ? kStages - 1 : stage - 1, next, page);
          advance();
          page = look_up();
        }
        cp_async_commit();
        const int p0 = unit_slot(a, at.span, at.u + i);
        float* w = a.new_scores ? a.weights + (((int64_t)at.b * c.kv_heads + kvh) * c.max_slots + p0) * a.group + g0 : nullptr;
        fold.template fold<WHOLE>(a, ring + stage * slot_bytes, valid_of[warp][stage], row_bytes,
                                  sizeof(T) == 2 ? (D + 15) / 16 : chunks, w, at.span.lo - p0, at.span.hi - p0, G, ps, qs);
        stage = stage == kStages - 1 ? 0 : stage + 1;
      }
      if (n == at.units) {
        const int64_t head = (int64_t)at.b * a.heads + h0;
        fold.end(static_cast<T*>(a.out) + head * D, nullptr, a.stats + head * 2, 0, G, D);
      } else {
        const int64_t to = (int64_t)(at.u > 0 ? 0 : TILE) * a.pieces + piece;
        fold.end(nullptr, a.parts + to * D, a.ml + to * 2, a.pieces, G, D);
        if (at.u > 0 && at.u + n == at.units) {
          ends = true;
          // it is the piece's first row, which the piece begins with unit at.u of
          const int64_t x = chunk_first(line.plan, cur.k.index) + first - at.u;
          if (lane == 0) a.joins[piece] = make_int4(at.b, at.r, piece_of(line.plan, WARPS, x), 0);
        }
      }
      left -= n;
      if (left > 0) at.step(a, rows, n);
    }
    if (lane == 0) a.ends[piece] = ends;
    if (!seamless) {
      coming = take();
      cp_async_wait<0>();
      __syncwarp();
      enter();
      start();
    }
    cur = coming;
    if (cur.k.b < 0 || *static_cast<volatile int*>(&s_abort)) break;
  }
  cp_async_wait<0>();
  // An answer may still be on its way: it is waited for. (The chunk that it names is then done by nobody: a call of which
  // a wait ran out leaves its outputs unfinished and the status set. Where the wait that ran out was one for `taken`, none
  // was asked for, and this takes its second; counting what was asked for cost healthy calls up to 2%.)
  if (s_abort && s_ask) mbar_drain(smem_u32(&answered), s_answers & 1);
}

// ---- short sequences: one kernel ------------------------------------------------------------------
// A cluster of CTAs a row: its warps have a run of the row's units each, the CTAs join their warps' parts in shared
// memory and then one another's through distributed shared memory, and each adds the weights of its own slots to
// the scores. Where the page table has room for kClusterUnits units a warp at most, this is one launch and two
// trips to memory after the lengths instead of two launches and six: 5.1 us instead of 11.5 us for one f32 token over
// 257 slots (16 query and 8 KV heads of 128), 10.4 instead of 19 us for 7 sequences of 1000 slots. Beyond about 8 units
// a warp the line is as fast, since it has all SMs.
constexpr int kMaxClusterCtas = 8;
constexpr int kClusterUnits = 8;
template <typename T, int DT, int TILE, bool WHOLE>
__global__ void __launch_bounds__(kWarpsOf<T, TILE> * 32, DT <= 128 ? 2 : 1)
    attention_cluster_kernel(const __grid_constant__ AttnArgs a) {
  using Fold = FoldOf<T, DT, TILE>;
  constexpr int U = Fold::U, WARPS = kWarpsOf<T, TILE>, THREADS = WARPS * 32;
  constexpr int VN = 16 / sizeof(T);
  __shared__ uint32_t valid_of[WARPS][kStages];
  __shared__ __align__(8) float mls[WARPS][TILE][2];
  __shared__ __align__(8) float cta_ml[TILE][2];
  __shared__ float2 stats[TILE];  // m, 1 / l of the row
  extern __shared__ __align__(16) char dyn[];
  const PagedView& c = a.cache;
  const int D = WHOLE ? DT : c.head_dim, tid = threadIdx.x, warp = tid >> 5;
  const int chunks = D / VN, row_bytes = row_chunks<T>(D) * 16, slot_bytes = 2 * U * row_bytes;
  char* ring = dyn + warp * kStages * slot_bytes;
  float* qs = reinterpret_cast<float*>(dyn + WARPS * kStages * slot_bytes) + warp * TILE * (D + U);
  float* ps = qs + TILE * D;
  const int C = (int)gridDim.x, rank = (int)blockIdx.x, rows = c.kv_heads * a.tiles;
  const int64_t row = blockIdx.y, b = row / rows;
  const int r = (int)(row - b * rows), kvh = r / a.tiles, g0 = (r - kvh * a.tiles) * TILE;
  const int G = min(TILE, a.group - g0), h0 = kvh * a.group + g0;
  zero_tails<T>(ring, kStages * 2 * U, D);
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  Fold fold;
  fold.load_q(a, b, h0, G, qs);
  const Span span = span_of(a, b);
  const int units = units_of(a, span), w = rank * WARPS + warp, all = C * WARPS;
  const int u0 = units * w / all, u1 = units * (w + 1) / all;
  fold.begin();
  int load = u0, page = -1;
  auto look_up = [&](int u) { return u < u1 ? look_up_page<U, WHOLE>(a, (int)b, span, unit_slot(a, span, u)) : -1; };
  auto send = [&](int stage, int pg) {
    if (load < u1) {
      load_rows<T, DT, U, WHOLE>(a, ring + stage * slot_bytes, &valid_of[warp][stage], span, unit_slot(a, span, load), kvh, pg);
      ++load;
    }
    cp_async_commit();
  };
  static_assert(kStages == 3, "the first units' pages are looked up together");
  {
    const int page0 = look_up(u0), page1 = look_up(u0 + 1);
    page = look_up(u0 + 2);
    send(0, page0);
    send(1, page1);
  }
  float* weights = a.new_scores ? a.weights + ((b * c.kv_heads + kvh) * c.max_slots) * a.group + g0 : nullptr;
  for (int u = u0, stage = 0; u < u1; ++u) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    send(stage == 0 ? kStages - 1 : stage - 1, page);
    page = look_up(load);
    const int p0 = unit_slot(a, span, u);
    fold.template fold<WHOLE>(a, ring + stage * slot_bytes, valid_of[warp][stage], row_bytes,
                              sizeof(T) == 2 ? (D + 15) / 16 : chunks, weights ? weights + (int64_t)p0 * a.group : nullptr,
                              span.lo - p0, span.hi - p0, G, ps, qs);
    stage = stage == kStages - 1 ? 0 : stage + 1;
  }
  // the warps' parts, each in its own ring
  cp_async_wait<0>();
  __syncwarp();
  fold.end(nullptr, reinterpret_cast<float*>(ring), &mls[warp][0][0], 1, G, D);
  __syncthreads();
  float* joined = reinterpret_cast<float*>(ring - warp * kStages * slot_bytes + slot_bytes);  // in the first ring's second stage
  for (int i = tid; i < G * D; i += THREADS) {
    const int g = i / D;
    float2 ml = make_float2(mls[0][g][0], mls[0][g][1]);
#pragma unroll
    for (int v = 1; v < WARPS; ++v) ml.x = fmaxf(ml.x, mls[v][g][0]);
    const float f = ml.x == -INFINITY ? 0.f : ml.x;
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int v = 0; v < WARPS; ++v) {
      const float e = ex2(mls[v][g][0] - f);
      o = fmaf(e, reinterpret_cast<const float*>(dyn + v * kStages * slot_bytes)[i], o);
      l = fmaf(e, mls[v][g][1], l);
    }
    joined[i] = o;
    if (i == g * D) {
      cta_ml[g][0] = ml.x;
      cta_ml[g][1] = l;
    }
  }
  cluster_sync_all();
  for (int i = rank * THREADS + tid; i < G * D; i += C * THREADS) {
    const int g = i / D;
    float m[kMaxClusterCtas], l[kMaxClusterCtas], o[kMaxClusterCtas];
#pragma unroll
    for (int k = 0; k < kMaxClusterCtas; ++k)
      if (k < C) {
        m[k] = ld_cluster_f32(&cta_ml[g][0], (unsigned)k);
        l[k] = ld_cluster_f32(&cta_ml[g][1], (unsigned)k);
        o[k] = ld_cluster_f32(joined + i, (unsigned)k);
      }
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMaxClusterCtas; ++k)
      if (k < C) M = fmaxf(M, m[k]);
    const float f = M == -INFINITY ? 0.f : M;
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int k = 0; k < kMaxClusterCtas; ++k)
      if (k < C) {
        const float e = ex2(m[k] - f);
        num = fmaf(e, o[k], num);
        den = fmaf(e, l[k], den);
      }
    static_cast<T*>(a.out)[(b * a.heads + h0) * D + i] = from_f32<T>(den == 0.f ? 0.f : num / den);
  }
  if (a.new_scores) {  // the heads are one tile
    if (tid < G) {
      float M = -INFINITY, den = 0.f;
      for (int k = 0; k < C; ++k) M = fmaxf(M, ld_cluster_f32(&cta_ml[tid][0], (unsigned)k));
      const float f = M == -INFINITY ? 0.f : M;
      for (int k = 0; k < C; ++k)
        den = fmaf(ex2(ld_cluster_f32(&cta_ml[tid][0], (unsigned)k) - f), ld_cluster_f32(&cta_ml[tid][1], (unsigned)k), den);
      stats[tid] = make_float2(f, den == 0.f ? 0.f : 1.f / den);
    }
    __syncthreads();
    const float* old = a.scores + (b * c.kv_heads + kvh) * c.max_slots;
    float* now = a.new_scores + (b * c.kv_heads + kvh) * c.max_slots;
    if (now != old)  // slots before the window keep theirs
      for (int p = rank * THREADS + tid; p < span.lo; p += C * THREADS) now[p] = old[p];
    const int first = max(span.lo, unit_slot(a, span, units * rank / C)), last = min(span.hi, unit_slot(a, span, units * (rank + 1) / C));
    for (int p = first + tid; p < last; p += THREADS) {
      float sum = 0.f;
      for (int g = 0; g < G; ++g) sum = fmaf(ex2(weights[(int64_t)p * a.group + g] - stats[g].x), stats[g].y, sum);
      now[p] = old[p] + sum;
    }
  }
  cluster_sync_all();  // no CTA leaves while another still reads its shared memory
}

// ---- finish ---------------------------------------------------------------------------------------
constexpr int kFinishThreads = 256;
constexpr int kFinishBlocks = kSms * 4;  // of joins, and about as many of scores
constexpr int kMaxJoins = 2 * kSms * kLevels * 4;  // a piece ends one at most

// (m, l) pairs joined; m of 0 weights is -inf, and l NaN where a score was NaN.
__device__ __forceinline__ float2 join(float2 x, float2 y) {
  const float m = fmaxf(x.x, y.x), f = m == -INFINITY ? 0.f : m;
  return make_float2(m, x.y * ex2(x.x - f) + y.y * ex2(y.x - f));
}

// The pieces in which a row ends that began in an earlier one, in order, to list; their number. By the block.
__device__ __forceinline__ int list_joins(const AttnArgs& a, uint16_t* list, int* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kRounds = (kMaxJoins + kFinishThreads * 16 - 1) / (kFinishThreads * 16);
  uint4 f[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {  // of 16 pieces a thread; those beyond the line's hold anything
    const int p0 = (r * kFinishThreads + tid) * 16;
    if (p0 < a.pieces) f[r] = *reinterpret_cast<const uint4*>(a.ends + p0);
  }
  const int pieces = a.plan->ctas * a.plan->levels * a.warps;
  int count = 0;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int p0 = (r * kFinishThreads + tid) * 16;
    const uint32_t w[4] = {f[r].x, f[r].y, f[r].z, f[r].w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (p0 + i < pieces && ((w[i / 4] >> (i % 4 * 8)) & 255) == 1) bits |= 1u << i;
    int incl = __popc(bits);
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += y;
    }
    if (lane == 31) red[warp] = incl;
    __syncthreads();
    int at = count + incl - __popc(bits);
    for (int w = 0; w < kFinishThreads / 32; ++w) {
      if (w < warp) at += red[w];
      count += red[w];
    }
    for (; bits; bits &= bits - 1) list[at++] = (uint16_t)(p0 + __ffs(bits) - 1);
    __syncthreads();
  }
  return count;
}

// Head g of the row that ends in piece `last`, `cols` columns of 4 values from col0, by the block: `cols`
// threads have the columns, and groups of them every so many-th part.
template <typename T>
__device__ __forceinline__ void join_head(const AttnArgs& a, int last, int g, int cols, int col0, float4* sums, float2* mls) {
  const int D = a.cache.head_dim, tid = threadIdx.x;
  const int4 row = a.joins[last];
  const int kvh = row.y / a.tiles, g0 = (row.y - kvh * a.tiles) * a.tile, first = row.z;
  // All the same for the block. Pieces of a chunk that nobody did, since a wait ran out, hold whatever the workspace
  // held before the call: nothing is read or written by what cannot be a row.
  if (row.x < 0 || row.x >= a.batch || row.y < 0 || row.y >= a.cache.kv_heads * a.tiles || first < 0 || first > last) return;
  if (g >= a.group - g0) return;
  const int lanes = kFinishThreads / cols, j = tid / cols, col = tid - j * cols, d = (col0 + col) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  float2 ml = make_float2(-INFINITY, 0.f);
  constexpr int kAtOnce = 4;  // parts whose loads are in flight together
  if (d < D)
    for (int p0 = first + j; p0 <= last; p0 += kAtOnce * lanes) {
      float2 x[kAtOnce];
      float4 v[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int p = p0 + i * lanes;
        const int64_t at = (int64_t)((p == first ? a.tile : 0) + g) * a.pieces + p;
        x[i] = make_float2(-INFINITY, 0.f);
        if (p <= last) {
          x[i] = *reinterpret_cast<const float2*>(a.ml + at * 2);
          v[i] = *reinterpret_cast<const float4*>(a.parts + at * D + d);
        }
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (x[i].x == -INFINITY) {  // nothing counted, or nothing written (l is 0); or, since a maximum passes NaN
          ml.y += x[i].y;           // over, all scores were NaN (l is NaN)
          continue;
        }
        const float m = fmaxf(ml.x, x[i].x), e0 = ex2(ml.x - m), e1 = ex2(x[i].x - m);
        ml = make_float2(m, ml.y * e0 + x[i].y * e1);
        s.x = s.x * e0 + v[i].x * e1;
        s.y = s.y * e0 + v[i].y * e1;
        s.z = s.z * e0 + v[i].z * e1;
        s.w = s.w * e0 + v[i].w * e1;
      }
    }
  // the groups' sums, by halves
  int n = 1;
  while (n < min(lanes, last - first + 1)) n *= 2;
  __syncthreads();
  sums[tid] = s;
  mls[tid] = ml;
  __syncthreads();
  for (n /= 2; n > 0; n /= 2) {
    if (j < n) {
      const float2 x = mls[tid + n * cols];
      const float4 v = sums[tid + n * cols];
      const float m = fmaxf(ml.x, x.x), f = m == -INFINITY ? 0.f : m, e0 = ex2(ml.x - f), e1 = ex2(x.x - f);
      ml = make_float2(m, ml.y * e0 + x.y * e1);
      s = make_float4(s.x * e0 + v.x * e1, s.y * e0 + v.y * e1, s.z * e0 + v.z * e1, s.w * e0 + v.w * e1);
      sums[tid] = s;
      mls[tid] = ml;
    }
    __syncthreads();
  }
  if (j == 0 && d < D) {
    const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
    T* out = static_cast<T*>(a.out) + ((int64_t)row.x * a.heads + kvh * a.group + g0 + g) * D + d;
    out[0] = from_f32<T>(s.x * inv);
    out[1] = from_f32<T>(s.y * inv);
    out[2] = from_f32<T>(s.z * inv);
    out[3] = from_f32<T>(s.w * inv);
  }
}

// The softmax weights of the slots of row (b, kvh) from `from`, every stride-th of them a thread's, added to
// the scores. VEC: heads that one load brings.
template <int VEC>
__device__ __forceinline__ void add_weights(const AttnArgs& a, const Plan& plan, int64_t row, int from, int stride,
                                            float2* st) {
  static_assert(kFinishThreads == 16 * kMaxTile, "16 threads a head");
  const PagedView& c = a.cache;
  const int tid = threadIdx.x;
  const int64_t b = row / c.kv_heads;
  const int kvh = (int)(row - b * c.kv_heads);
  const Span sp = span_of(a, b);
  if (sp.hi == 0) return;
  const int units = units_of(a, sp);
  const float* old = a.scores + row * c.max_slots;
  float* now = a.new_scores + row * c.max_slots;
  if (now != old)  // slots before the window keep theirs
    for (int p = from + tid; p < sp.lo; p += stride) now[p] = old[p];
  for (int t = 0; t < a.tiles; ++t) {
    const int t0 = t * a.tile, G = min(a.tile, a.group - t0);
    const int64_t x = a.seq_first[b] + (int64_t)(kvh * a.tiles + t) * units;
    const int first = piece_of(plan, a.warps, x), last = piece_of(plan, a.warps, x + units - 1);
    __syncthreads();
    if (first == last) {
      const float* s = a.stats + (b * a.heads + kvh * a.group + t0) * 2;
      if (tid < G) st[tid] = make_float2(s[2 * tid], s[2 * tid + 1]);
    } else {
      const int g = min(tid / 16, G - 1), j = tid & 15;
      float2 ml = make_float2(-INFINITY, 0.f);
#pragma unroll 4
      for (int p = first + j; p <= last; p += 16) {
        ml = join(ml, *reinterpret_cast<const float2*>(a.ml + ((int64_t)((p == first ? a.tile : 0) + g) * a.pieces + p) * 2));
      }
      for (int off = 8; off > 0; off >>= 1)
        ml = join(ml, make_float2(__shfl_xor_sync(0xffffffffu, ml.x, off), __shfl_xor_sync(0xffffffffu, ml.y, off)));
      if (j == 0 && tid / 16 < G) st[g] = make_float2(ml.x == -INFINITY ? 0.f : ml.x, ml.y == 0.f ? 0.f : 1.f / ml.y);
    }
    __syncthreads();
    const float* w = a.weights + row * c.max_slots * a.group + t0;
    constexpr int kAtOnce = 4;  // slots of a thread whose loads are in flight together
    for (int p0 = sp.lo + from + tid; p0 < sp.hi; p0 += kAtOnce * stride) {
      float was[kAtOnce], sum[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int p = p0 + k * stride;
        was[k] = p < sp.hi ? (t == 0 ? old[p] : now[p]) : 0.f;
        sum[k] = 0.f;
      }
      for (int g = 0; g < G; g += VEC) {
        float y[kAtOnce][VEC];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int p = min(p0 + k * stride, sp.hi - 1);
          const float* src = w + (int64_t)p * a.group + g;
          if constexpr (VEC == 4) *reinterpret_cast<float4*>(y[k]) = *reinterpret_cast<const float4*>(src);
          else if constexpr (VEC == 2) *reinterpret_cast<float2*>(y[k]) = *reinterpret_cast<const float2*>(src);
          else y[k][0] = src[0];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float2 ml = st[g + i];
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) sum[k] = fmaf(ex2(y[k][i] - ml.x), ml.y, sum[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k)
        if (p0 + k * stride < sp.hi) now[p0 + k * stride] = was[k] + sum[k];
    }
  }
}

// kFinishBlocks blocks, the even ones of the first where there are scores too: joins. The others: scores, `pieces`
// blocks a row.
template <typename T, int VEC>
__global__ void __launch_bounds__(kFinishThreads, 4)
    attention_finish_kernel(const __grid_constant__ AttnArgs a, int pieces) {
  __shared__ float4 sums[kFinishThreads];
  __shared__ float2 mls[kFinishThreads];
  __shared__ Plan plan;
  __shared__ uint16_t list[kMaxJoins];
  __shared__ int red[kFinishThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int D = a.cache.head_dim, tid = threadIdx.x;
  const int scorers = gridDim.x - kFinishBlocks, both = 2 * min(scorers, kFinishBlocks);
  const int index = (int)blockIdx.x < both ? blockIdx.x / 2 : blockIdx.x - both / 2;
  if ((int)blockIdx.x < both ? (blockIdx.x & 1) == 0 : scorers < kFinishBlocks) {
    const int n = list_joins(a, list, red);
    // A task is a head's columns. Few rows have many parts each: their columns are spread over more blocks,
    // whose threads then have more groups for the parts.
    const int G = min(a.tile, a.group), all = D / 4;
    int cols = 2;
    while (cols < all) cols *= 2;
    while (cols > 4 && n * G * ((all + cols / 2 - 1) / (cols / 2)) <= kFinishBlocks) cols /= 2;
    const int splits = (all + cols - 1) / cols, tasks = n * G * splits;
    for (int task = index; task < tasks; task += kFinishBlocks) {
      const int head = task / splits, row = head / G;
      join_head<T>(a, list[row], head - row * G, cols, (task - head * splits) * cols, sums, mls);
    }
    // sequences without slots give zeros
    for (int64_t b = index; b < a.batch; b += kFinishBlocks)
      if (span_of(a, b).hi == 0)
        for (int i = tid; i < a.heads * D; i += kFinishThreads) static_cast<T*>(a.out)[b * a.heads * D + i] = from_f32<T>(0.f);
  } else {
    if (tid == 0) plan = *a.plan;
    __syncthreads();
    const int64_t row = index / pieces;
    add_weights<VEC>(a, plan, row, (int)(index - row * pieces) * kFinishThreads, pieces * kFinishThreads, mls);
  }
}

namespace {

int head_tile(const tq4_paged_desc& d, int heads) {
  const int group = heads / d.kv_heads;
  if (d.dtype == TQ4_F32) return group >= 5 ? 8 : group >= 3 ? 4 : group;
  return group > 8 ? 16 : 8;
}

// How a call is cut, from what the host knows of it.
struct Shape {
  int tile, tiles, unit, unit_log2, warps, ctas, levels;
  int64_t grid;  // as many chunks as sequences that fill the page table would give
};
Shape shape_of(const tq4_paged_desc& d, int heads, int64_t batch) {
  Shape s;
  const int group = heads / d.kv_heads;
  s.tile = head_tile(d, heads);
  s.tiles = (group + s.tile - 1) / s.tile;
  // the folds' U and the kernels' warps and residence
  s.unit = d.dtype == TQ4_F32 ? (d.head_dim <= 64 ? 16 : 8) : (d.head_dim <= 64 ? 32 : 16);
  s.unit_log2 = s.unit == 8 ? 3 : s.unit == 16 ? 4 : 5;
  s.warps = d.dtype == TQ4_F32 && s.tile == 8 ? 3 : 4;
  s.ctas = d.head_dim <= 128 ? 2 * kSms : kSms;
  const int64_t slots = (int64_t)d.max_pages * d.page_size;
  const int64_t most = batch * d.kv_heads * s.tiles * ((slots + s.unit - 1) / s.unit + 1);
  s.levels = 1;
  for (int64_t left = most / s.ctas; s.levels < kLevels && left >= 2 * kMinChunk; ++s.levels)
    left = std::max<int64_t>(left * 3 / 8, kMinChunk);
  s.grid = s.levels > 1 ? (int64_t)s.ctas * s.levels : std::min<int64_t>(s.ctas, (most + s.warps - 1) / s.warps);
  return s;
}

// CTAs of a row for the cluster kernel; 0 where the line's kernels are to be used. The cluster kernel takes rows
// that do not fill the SMs twice over, with room in the page table (or the window) for few units a warp, and with
// all heads of a KV head in one row where there are scores.
int cluster_size(const tq4_paged_desc& d, const Shape& s, int64_t batch, int64_t window, bool with_scores) {
  const int64_t rows = batch * d.kv_heads * s.tiles;
  int64_t slots = (int64_t)d.max_pages * d.page_size;
  if (window > 0) slots = std::min(slots, window + s.unit);
  const int64_t units = (slots + s.unit - 1) / s.unit;
  if (rows > s.ctas || (with_scores && s.tiles > 1)) return 0;
  int c = 1;
  while (c < kMaxClusterCtas && rows * c * 2 <= s.ctas && units > (int64_t)c * s.warps) c *= 2;
  return units <= (int64_t)c * s.warps * kClusterUnits ? c : 0;
}

// Offsets of the workspace's parts, in bytes, each a multiple of 16. What the cluster kernel takes whatever the
// window needs none but the scores'.
struct Workspace {
  int64_t seq_first, ends, joins, stats, ml, parts, weights, bytes;
};
Workspace workspace_of(const tq4_paged_desc& d, int heads, int64_t batch, bool with_scores) {
  auto up = [](int64_t n) { return (n + 15) / 16 * 16; };
  const Shape s = shape_of(d, heads, batch);
  const bool line = cluster_size(d, s, batch, 0, with_scores) == 0;
  const int64_t slots = s.grid * s.warps * 2 * s.tile;
  Workspace w{};
  if (!line) {
    w.bytes = with_scores ? up(batch * heads * (int64_t)d.max_pages * d.page_size * 4) : 0;
    return w;
  }
  w.seq_first = up(sizeof(Plan));
  w.ends = w.seq_first + up(batch * 8);
  w.joins = w.ends + up(s.grid * s.warps);
  w.stats = w.joins + s.grid * s.warps * 16;
  w.ml = w.stats + up(batch * heads * 2 * 4);
  w.parts = w.ml + up(slots * 2 * 4);
  w.weights = w.parts + up(slots * d.head_dim * 4);
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
tq4_status launch_cluster(const AttnArgs& a, int c, cudaStream_t st) {
  const bool whole = a.cache.head_dim == DT;
  const auto kern = whole ? attention_cluster_kernel<T, DT, TILE, true> : attention_cluster_kernel<T, DT, TILE, false>;
  static std::atomic<uint64_t> set[2];  // per device, per instantiation
  TQ4_CUDA(set_smem_limit_once(kern, part_smem<T, DT, TILE>(DT), set[whole]));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c, (unsigned)(a.batch * a.cache.kv_heads * a.tiles));
  cfg.blockDim = dim3(a.warps * 32);
  cfg.dynamicSmemBytes = part_smem<T, DT, TILE>(a.cache.head_dim);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  TQ4_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  return TQ4_OK;
}

template <typename T, int DT, int TILE>
tq4_status launch_part(AttnArgs& a, int64_t grid, cudaStream_t st) {
  if (a.unit != FoldOf<T, DT, TILE>::U || a.warps != kWarpsOf<T, TILE>) {
    set_error("tq4_paged_attention: the call was cut for other kernels");
    return TQ4_ERR_UNSUPPORTED;
  }
  if (a.cluster) return launch_cluster<T, DT, TILE>(a, a.cluster, st);
  const bool whole = a.cache.head_dim == DT;
  const auto kern = whole ? attention_part_kernel<T, DT, TILE, true> : attention_part_kernel<T, DT, TILE, false>;
  static std::atomic<uint64_t> set[2];  // per device, per instantiation
  TQ4_CUDA(set_smem_limit_once(kern, part_smem<T, DT, TILE>(DT), set[whole]));
  TQ4_CUDA(launch_pdl(kern, dim3((unsigned)grid), dim3(a.warps * 32), part_smem<T, DT, TILE>(a.cache.head_dim), st, a));
  return TQ4_OK;
}

template <typename T, int TILE>
tq4_status launch_width(AttnArgs& a, int64_t grid, cudaStream_t st) {
  const int D = a.cache.head_dim;
  if (D <= 64) return launch_part<T, 64, TILE>(a, grid, st);
  if (D <= 128) return launch_part<T, 128, TILE>(a, grid, st);
  return launch_part<T, 256, TILE>(a, grid, st);
}

template <typename T>
tq4_status launch_attention(AttnArgs& a, int64_t grid, cudaStream_t st) {
  if constexpr (sizeof(T) == 4) {
    switch (a.tile) {
      case 1: TQ4_TRY((launch_width<T, 1>(a, grid, st))); break;
      case 2: TQ4_TRY((launch_width<T, 2>(a, grid, st))); break;
      case 4: TQ4_TRY((launch_width<T, 4>(a, grid, st))); break;
      default: TQ4_TRY((launch_width<T, 8>(a, grid, st))); break;
    }
  } else {
    if (a.tile == 8) TQ4_TRY((launch_width<T, 8>(a, grid, st)));
    else TQ4_TRY((launch_width<T, 16>(a, grid, st)));
  }
  if (a.cluster) return TQ4_OK;
  const auto finish = a.group % 4 == 0   ? attention_finish_kernel<T, 4>
                      : a.group % 2 == 0 ? attention_finish_kernel<T, 2>
                                         : attention_finish_kernel<T, 1>;
  const int64_t rows = a.batch * a.cache.kv_heads;
  const int pieces = (int)std::min<int64_t>(std::max<int64_t>(1, 2 * kFinishBlocks / rows),
                                            (a.cache.max_slots + kFinishThreads - 1) / kFinishThreads);
  const int64_t blocks = kFinishBlocks + (a.new_scores ? rows * pieces : 0);
  TQ4_CUDA(launch_pdl(finish, dim3((unsigned)blocks), dim3(kFinishThreads), 0, st, a, pieces));
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
  if (!q || !lengths || !out || (scores != nullptr) != (new_scores != nullptr)) {
    set_error("tq4_paged_attention: null q, lengths or out, or only one of scores and new_scores");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (window < 0 || q_stride < (int64_t)heads * d.head_dim) {
    set_error("tq4_paged_attention: window %lld below 0, or q_stride %lld below heads * head_dim", (long long)window,
              (long long)q_stride);
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  const int64_t out_values = batch * heads * d.head_dim, size = dtype_size(d.dtype);
  if (overlaps(q, ((batch - 1) * q_stride + (int64_t)heads * d.head_dim) * size, out, out_values * size)) {
    set_error("tq4_paged_attention: out overlaps q");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  const int64_t score_bytes = batch * d.kv_heads * (int64_t)d.max_pages * d.page_size * 4;
  if (scores != new_scores && overlaps(scores, score_bytes, new_scores, score_bytes)) {
    set_error("tq4_paged_attention: new_scores overlaps scores and is not the same buffer");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  if (window >= (int64_t)d.max_pages * d.page_size) window = 0;  // no sequence reaches it
  const Workspace ws = workspace_of(d, heads, batch, scores != nullptr);
  if (workspace_bytes < ws.bytes || !aligned16(workspace) || (ws.bytes > 0 && !workspace)) {
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
  const Shape shape = shape_of(d, heads, batch);
  a.tile = shape.tile;
  a.tiles = shape.tiles;
  a.unit = shape.unit;
  a.unit_log2 = shape.unit_log2;
  a.warps = shape.warps;
  a.ctas = shape.ctas;
  a.levels = shape.levels;
  a.q_even = (reinterpret_cast<uintptr_t>(q) & 3) == 0 && (q_stride & 1) == 0;
  a.scale2 = scale * kLog2e;
  a.scores = scores;
  a.new_scores = new_scores;
  char* w = static_cast<char*>(workspace);
  a.plan = reinterpret_cast<Plan*>(w);
  a.seq_first = reinterpret_cast<int64_t*>(w + ws.seq_first);
  a.ends = reinterpret_cast<uint8_t*>(w + ws.ends);
  a.joins = reinterpret_cast<int4*>(w + ws.joins);
  a.stats = reinterpret_cast<float*>(w + ws.stats);
  a.ml = reinterpret_cast<float*>(w + ws.ml);
  a.pieces = (int)shape.grid * shape.warps;
  a.parts = reinterpret_cast<float*>(w + ws.parts);
  a.weights = reinterpret_cast<float*>(w + ws.weights);
  a.cluster = cluster_size(d, shape, batch, window, scores != nullptr);
  if (batch * d.kv_heads * a.tiles > ((int64_t)1 << 30)) {
    set_error("tq4_paged_attention: more than 2^30 rows of sequences and KV heads");
    return TQ4_ERR_INVALID_ARGUMENT;
  }
  DeviceGuard guard(cache->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (d.dtype) {
    case TQ4_F16: return launch_attention<__half>(a, shape.grid, st);
    case TQ4_BF16: return launch_attention<__nv_bfloat16>(a, shape.grid, st);
    default: return launch_attention<float>(a, shape.grid, st);
  }
}

}  // extern "C"
