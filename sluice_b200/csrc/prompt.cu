// The prompt pass's small operators: the KV block planner (block tables and
// slot maps from request lengths) and rotary positions.
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

// ------------------------------------------------------------ block planner
// Request r holds held = ceil(context / bs) blocks and needs
// need = ceil((context + new) / bs). With take = need - held and
// off = the sum of take over the requests before it, its i-th new block is
// free[(head + off + i) mod N]. Token i of the request sits at position
// context + i, in slot block(position / bs) * bs + position mod bs.
//
// Every CTA makes the same scan over the requests in shared memory and then
// fills its share of the tables and maps. A new block's id is read from the
// free ring, not from the table, so no CTA waits for another's table writes;
// the ring's range is read by all and written by none of a launch of several
// CTAs that updates it in place (plan_range_kernel then writes it).
//
// Bound by latency: the lengths, the scan, a search and a table entry follow one
// another. Eight single tokens take 3.8 to 4.4 us, 256 take 4.5, 72 000 rows 6.5,
// 2.2 million (17 MB, 2.6 us at copy bandwidth) 16; with a row a lane at a time and
// one warp for the table the last two took 35 and 40 us.
constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxRequests = 8192;
constexpr int kPlanFew = 2;      // blocks that a lane writes by itself
constexpr int kPlanChunk = 128;  // consecutive rows that a warp fills in a turn, four a lane

struct PlanArgs {
  const int32_t* context;
  const int32_t* fresh;
  int B, bs, shift, width, N;  // shift: log2 of bs, -1 where it is no power of two
  int64_t T, Tk;
  int32_t* table;
  int64_t ld_table;
  const int32_t* free_blocks;
  const int64_t* range;
  int64_t* range_out;
  int32_t* cu_new;
  int32_t* cu_total;
  int64_t* positions;
  int64_t* slots;
  int64_t* kv_slots;
  int32_t* status;
  int write_range;
};

struct Lengths {
  int context, fresh, held, take;
  bool invalid, refused;
};

// x / block size, and the blocks that x >= 0 rows take. (Positions are unsigned:
// a refused request's may pass 31 bits.)
__device__ __forceinline__ int block_index(const PlanArgs& a, unsigned x) {
  return static_cast<int>(a.shift >= 0 ? x >> a.shift : x / static_cast<unsigned>(a.bs));
}
__device__ __forceinline__ int blocks_of(const PlanArgs& a, int x) {
  const unsigned up = static_cast<unsigned>(x) + static_cast<unsigned>(a.bs) - 1u;
  return static_cast<int>(a.shift >= 0 ? up >> a.shift : up / static_cast<unsigned>(a.bs));
}

// One request's lengths, made safe: negative ones count as zero, and a
// request that does not fit its table row takes nothing.
__device__ __forceinline__ Lengths plan_lengths(const PlanArgs& a, int r) {
  Lengths l;
  l.context = a.context[r];
  l.fresh = a.fresh[r];
  l.invalid = l.context < 0 || l.fresh < 0;
  l.context = max(l.context, 0);
  l.fresh = max(l.fresh, 0);
  const int64_t total = static_cast<int64_t>(l.context) + l.fresh;
  // (a total past 31 bits fits no table row: more blocks than it has entries,
  // or entries past its memory)
  const bool huge = total > 0x7fffffff;
  int held = blocks_of(a, l.context);
  const int need = huge ? held : blocks_of(a, static_cast<int>(total));
  l.refused = need > a.width || huge;
  l.invalid |= held > a.width || huge;
  // (without a ring every block is in the table)
  if (a.free_blocks == nullptr) held = need;
  l.held = held;
  l.take = l.refused ? 0 : need - held;
  return l;
}

__device__ __forceinline__ int saturated(int64_t v) {
  return static_cast<int>(v < 0x7fffffff ? v : 0x7fffffff);
}

// Inclusive scan of three sums over the CTA (each warp by shuffles, then
// the warps' totals); `tot` receives the CTA's sums.
__device__ __forceinline__ void scan3(int64_t (&v)[3], int64_t (*warp_sum)[32], int64_t (&tot)[3]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v[k], o);
      if (lane >= o) v[k] += u;
    }
    if (lane == 31) warp_sum[k][warp] = v[k];
  }
  __syncthreads();
  if (warp < 3) {
    int64_t s = lane < nw ? warp_sum[warp][lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    warp_sum[warp][lane] = s;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (warp > 0) v[k] += warp_sum[k][warp - 1];
    tot[k] = warp_sum[k][nw - 1];
  }
  __syncthreads();
}

// The request that row t of a packed batch belongs to, known to lie in
// [lo, hi]: the last r with cu[r] <= t.
__device__ __forceinline__ int find_request(const int* cu, int t, int lo, int hi) {
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kv_blocks_kernel(PlanArgs a) {
  extern __shared__ int plan_sm[];
  __shared__ int64_t warp_sum[3][32];
  __shared__ int s_invalid, s_short, s_end;
  int* cu_new = plan_sm;                 // [B + 1]
  int* cu_total = cu_new + a.B + 1;      // [B + 1]
  int* off = cu_total + a.B + 1;         // [B] blocks taken before, -1: refused
  int* cached = off + a.B;               // [B] context (the sums above may be cut off)
  const int tid = threadIdx.x, lane = tid & 31;
  if (tid == 0) {
    s_invalid = s_short = s_end = 0;
    cu_new[0] = cu_total[0] = 0;
  }
  sl::pdl_wait();
  sl::pdl_trigger();
  const bool ring = a.free_blocks != nullptr;
  int64_t head = ring ? a.range[0] : 0;
  int64_t avail = ring ? a.range[1] - head : 0;
  const bool bad_range = avail < 0 || avail > a.N || head < 0;
  if (bad_range) head = avail = 0;
  __syncthreads();

  // the scan: rows before each request and blocks taken before it
  int64_t carry[3] = {0, 0, 0};
  for (int r0 = 0; r0 < a.B; r0 += blockDim.x) {
    const int r = r0 + tid;
    Lengths l = {};
    if (r < a.B) l = plan_lengths(a, r);
    int64_t v[3] = {l.fresh, static_cast<int64_t>(l.context) + l.fresh, l.take}, tot[3];
    scan3(v, warp_sum, tot);
    if (r < a.B) {
      const int64_t end = carry[2] + v[2];
      // a request is served when its blocks end inside the free range, or
      // when it needs none
      const bool short_of = l.take > 0 && end > avail;
      cu_new[r + 1] = saturated(carry[0] + v[0]);
      cu_total[r + 1] = saturated(carry[1] + v[1]);
      off[r] = l.refused || short_of ? -1 : saturated(end - l.take);
      cached[r] = l.context;
      if (l.take > 0 && !short_of) atomicMax(&s_end, saturated(end));
      if (l.invalid) s_invalid = 1;
      if (l.refused || short_of) s_short = 1;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) carry[k] += tot[k];
  }
  __syncthreads();
  // more rows than the outputs hold, or than 32-bit offsets count
  const bool over = carry[0] > a.T || carry[1] > 0x7fffffff || (a.Tk > 0 && carry[1] > a.Tk);

  const int gwarp = (blockIdx.x * blockDim.x + tid) >> 5, nwarps = (gridDim.x * blockDim.x) >> 5;
  // the i-th free block: head and i are at most the ring's size
  const int64_t ring_at = ring ? head % a.N : 0;
  auto new_block = [&](int i) -> const int32_t* {
    int64_t at = ring_at + i;
    if (at >= a.N) at -= a.N;
    return a.free_blocks + at;
  };
  // where the cache block of a row is found (nullptr: the row has none)
  auto block_at = [&](int r, int context, unsigned pos) -> const int32_t* {
    const int blk = block_index(a, pos), o = off[r];
    // a refused request's new rows have no slot, even inside its last block
    if (o < 0 && pos >= static_cast<unsigned>(context)) return nullptr;
    // without a ring every block is in the table, or nowhere: a context may
    // reach past its table row
    if (!ring || blk < blocks_of(a, context))
      return blk < a.width ? a.table + r * a.ld_table + blk : nullptr;
    return new_block(o + (blk - blocks_of(a, context)));
  };
  // rows of a packed batch, consecutive ones per warp and turn (four a lane, or
  // fewer where that would leave warps without any): a lane's are looked up
  // together, so that their loads overlap
  constexpr int kEach = kPlanChunk / 32;
  auto fill = [&](const int* cu, int64_t rows, bool all_rows) {
    const int used = cu[a.B];
    const int64_t turn = static_cast<int64_t>(nwarps) * 32;
    const int each = rows >= kEach * turn ? kEach : static_cast<int>((rows + turn - 1) / turn);
    const int chunk = 32 * each;
    for (int64_t c0 = static_cast<int64_t>(gwarp) * chunk; c0 < rows;
         c0 += static_cast<int64_t>(nwarps) * chunk) {
      int lo = 0, hi = 0;
      if (c0 < used) {
        lo = find_request(cu, static_cast<int>(c0), 0, a.B - 1);
        const int64_t last = min(c0 + chunk, min(rows, static_cast<int64_t>(used))) - 1;
        hi = find_request(cu, static_cast<int>(last), lo, a.B - 1);
      }
      unsigned pos[kEach];
      int block[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int64_t t = c0 + lane + 32 * i;
        pos[i] = ~0u;
        block[i] = -1;
        if (i < each && t < rows && t < used) {
          const int r = find_request(cu, static_cast<int>(t), lo, hi);
          const int context = cached[r];
          pos[i] = static_cast<unsigned>(static_cast<int>(t) - cu[r]) +
              (all_rows ? 0u : static_cast<unsigned>(context));
          const int32_t* at = block_at(r, context, pos[i]);
          if (at != nullptr) block[i] = *at;
        }
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int64_t t = c0 + lane + 32 * i;
        if (i >= each || t >= rows) continue;
        const int64_t slot = block[i] < 0 ? -1
            : static_cast<int64_t>(block[i]) * a.bs +
                (pos[i] - static_cast<unsigned>(block_index(a, pos[i])) * static_cast<unsigned>(a.bs));
        if (all_rows) {
          a.kv_slots[t] = slot;
        } else {
          a.positions[t] = pos[i] == ~0u ? -1 : static_cast<int64_t>(pos[i]);
          a.slots[t] = slot;
        }
      }
    }
  };
  fill(cu_new, a.T, false);
  if (a.kv_slots != nullptr) fill(cu_total, a.Tk, true);

  // the table rows of the requests that take blocks: a lane looks at each of
  // the warp's (nwarps apart) and writes a few blocks by itself, the warp writes
  // more (1000 requests that take one block each: 9.3 us, row after row 16.7)
  for (int r0 = gwarp; r0 < a.B; r0 += 32 * nwarps) {
    const int r = r0 + nwarps * lane;
    Lengths l = {};
    if (r < a.B) l = plan_lengths(a, r);
    const int o = r < a.B ? off[r] : -1;
    const bool few = l.take <= kPlanFew;
    if (few && o >= 0) {
      int32_t* row = a.table + r * a.ld_table + l.held;
      int id[kPlanFew];
#pragma unroll
      for (int i = 0; i < kPlanFew; ++i)
        if (i < l.take) id[i] = *new_block(o + i);
#pragma unroll
      for (int i = 0; i < kPlanFew; ++i)
        if (i < l.take) row[i] = id[i];
    }
    for (unsigned takers = __ballot_sync(0xffffffffu, o >= 0 && !few); takers;
         takers &= takers - 1) {
      const int w = __ffs(takers) - 1;
      const int first = __shfl_sync(0xffffffffu, o, w), n = __shfl_sync(0xffffffffu, l.take, w);
      int32_t* row = a.table + (r0 + nwarps * w) * a.ld_table + __shfl_sync(0xffffffffu, l.held, w);
      for (int i = lane; i < n; i += 32) row[i] = *new_block(first + i);
    }
  }
  if (blockIdx.x == 0) {
    // offsets that a reader may follow: never past the rows that were filled
    const int cap = saturated(a.T), cap_k = a.Tk > 0 ? saturated(a.Tk) : 0x7fffffff;
    for (int r = tid; r <= a.B; r += blockDim.x) {
      a.cu_new[r] = min(cu_new[r], cap);
      a.cu_total[r] = min(cu_total[r], cap_k);
    }
    if (tid == 0) {
      a.status[0] = s_invalid || bad_range || over ? SL_KV_PLAN_BAD_INPUT
                    : s_short                      ? SL_KV_PLAN_NO_BLOCKS
                                                   : SL_KV_PLAN_OK;
      a.status[1] = s_end;
      if (ring && a.write_range) {
        const int64_t first = a.range[0], tail = a.range[1];
        a.range_out[0] = first + s_end;
        a.range_out[1] = tail;
      }
    }
  }
}

// The free range of a plan that several CTAs read, moved on in place.
__global__ void plan_range_kernel(int64_t* range, const int32_t* status) {
  sl::pdl_wait();
  sl::pdl_trigger();
  range[0] += status[1];
}

// ------------------------------------------------------------------- rotary
// A pair (a, b) of a head at position p becomes (a cos t - b sin t,
// b cos t + a sin t) times a factor, t = p * freq. The angle is formed in
// turns, p * (freq / 2 pi), in 64 bits, whole turns taken off there, and only
// the rest (at most half a turn) goes to 32 bits, so a position of a million
// keeps as many bits of its phase as position one. Pairs are adjacent columns
// (interleaved) or columns rot / 2 apart (half).
constexpr int kRotThreads = 128;
constexpr int kRotMaxPairs = 256;

struct RotTensor {
  const void* x;
  void* y;
  int64_t xs, xh, ys, yh;  // strides of a token and a head, in elements
  int heads, offset, copied;  // copied: columns that are not rotated, where they are written
  int units;               // units of a head: its rotated ones, then the copied
  uint32_t units_mul;      // index / units == (index * units_mul) >> 32
};

struct RotArgs {
  const int64_t* positions;
  const double* turns;  // [rot / 2] turns per position
  float factor;
  int T, rot, per_cta, rot_units;
  float inv_items;      // 1 / units of a token, of all its heads
  RotTensor t[2];
};

template <typename E>
__device__ __forceinline__ float to_f(E v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename E>
__device__ __forceinline__ E from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

template <typename E, int V>
struct alignas(sizeof(E) * V) RotVec {
  E e[V];
};

// (products and sums are written out, so that every form of the kernel rounds
// alike.) A unit is two vectors of V columns, rot / 2 columns apart, V pairs:
// element k of both (half), or the neighbours within each (interleaved; with V =
// 1 a unit is two neighbours). A vector is 32 bytes where the sizes, strides and
// addresses allow it.
//
// Bound by the rows' bytes: enough of them have to be in flight (32-byte vectors,
// 8 CTAs of one unit a thread per SM: 49 us for 16384 rows of 36 heads of 128
// columns of bf16, 6.15 TB/s; 6 CTAs 51, 9 CTAs 51; 16-byte vectors 53, rows that
// allow 8, 4 and 2 bytes 76, 104 and 155, so the widest that fits is taken; in
// fp32 91, 6.6 TB/s). A CTA takes a few tokens, so that there are many of them (3
// tokens; 8 take 52). Columns that are not rotated go two vectors a unit too (one
// a unit: 4099 rows with 32 of 128 columns rotated 13.5 us, two 11.2). The first
// rows are asked for before the angles are formed.
template <typename E, int V, bool kInterleaved>
__global__ void __launch_bounds__(kRotThreads, V * sizeof(E) == 32   ? 8
                                               : V * sizeof(E) == 16 ? 10
                                                                     : 12) rotary_kernel(RotArgs a) {
  // (cos, sin) * factor of each token, [pair within a unit][unit]: lanes of
  // neighbouring units read neighbouring words
  extern __shared__ float2 cs[];
  __shared__ int s_skip[32];
  using Vec = RotVec<E, V>;
  sl::pdl_wait();
  sl::pdl_trigger();
  const int half = a.rot >> 1;
  // interleaved vectors hold whole pairs, or (V = 1) an element of one each
  constexpr bool kWithin = kInterleaved && V > 1;
  const int to_hi = kInterleaved && V == 1 ? 1 : half;  // from a unit's first vector to its second
  const int t0 = blockIdx.x * a.per_cta;
  const int nt = min(a.per_cta, a.T - t0);
  const int nq = a.t[0].heads * a.t[0].units, n = nq + a.t[1].heads * a.t[1].units;
  // the unit of a thread's turn
  Vec lo, hi;
  E* dst;
  int pair;   // first pair's place in cs, -1: not rotated
  int to;     // from the first vector to the second, 0: there is none
  int token;  // -1: no unit
  auto load = [&](int i) {
    token = -1;
    if (i >= nt * n) return;
    // i / n (exact: a CTA of several tokens has at most 2^12 items)
    const int t = a.per_cta == 1 ? 0 : static_cast<int>((i + 0.5f) * a.inv_items);
    const int w = i - t * n;
    const RotTensor& x = w < nq ? a.t[0] : a.t[1];
    const int idx = w < nq ? w : w - nq;
    const int head = x.units == 1 ? idx
                                  : static_cast<int>(__umulhi(static_cast<uint32_t>(idx), x.units_mul));
    const int unit = idx - head * x.units;
    int col;
    if (unit < a.rot_units) {
      col = x.offset + unit * (kInterleaved && V == 1 ? 2 : V);
      pair = t * half + unit;
      to = to_hi;
    } else {
      // columns that are not rotated, two vectors a unit: those before the
      // rotated ones, then those behind them
      const int c = (unit - a.rot_units) * (2 * V);
      col = c < x.offset ? c : c + a.rot;
      pair = -1;
      to = c + V >= x.copied ? 0 : c + V == x.offset ? V + a.rot : V;
    }
    token = t;
    const E* src = static_cast<const E*>(x.x) + (t0 + t) * x.xs + head * x.xh + col;
    dst = static_cast<E*>(x.y) + (t0 + t) * x.ys + head * x.yh + col;
    lo = *reinterpret_cast<const Vec*>(src);
    if (to != 0) hi = *reinterpret_cast<const Vec*>(src + to);
  };
  // the first rows are on their way while the angles are formed
  load(threadIdx.x);
  for (int i = threadIdx.x; i < nt * half; i += kRotThreads) {
    const int t = i / half, j = i - t * half;
    const int64_t p = a.positions[t0 + t];
    const double turns = static_cast<double>(p) * a.turns[j];
    float s, c;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
    // pair j's place in its unit, and the unit
    constexpr int kIn = V > 1 ? V / 2 : 1;
    const int back = kWithin && j >= half / 2 ? half / 2 : 0;
    const int k = kWithin ? (back ? kIn : 0) + (j - back) % kIn : j % V;
    const int unit = kWithin ? (j - back) / kIn : j / V;
    cs[t * half + k * a.rot_units + unit] = make_float2(c * a.factor, s * a.factor);
    if (j == 0) s_skip[t] = p < 0;
  }
  __syncthreads();
  for (int i = threadIdx.x;;) {
    if (token >= 0) {
      if (pair >= 0 && !s_skip[token]) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float2 c = cs[pair + k * a.rot_units];
          constexpr int kIn = V > 1 ? V / 2 : 1;  // pairs of one vector
          E& e0 = !kWithin ? lo.e[k] : k < kIn ? lo.e[2 * k % V] : hi.e[2 * k % V];
          E& e1 = !kWithin ? hi.e[k] : k < kIn ? lo.e[(2 * k + 1) % V] : hi.e[(2 * k + 1) % V];
          const float x0 = to_f(e0), x1 = to_f(e1);
          e0 = from_f<E>(fmaf(x0, c.x, -__fmul_rn(x1, c.y)));
          e1 = from_f<E>(fmaf(x1, c.x, __fmul_rn(x0, c.y)));
        }
      }
      *reinterpret_cast<Vec*>(dst) = lo;
      if (to != 0) *reinterpret_cast<Vec*>(dst + to) = hi;
    }
    i += kRotThreads;
    if (i >= nt * n) break;
    load(i);
  }
}

template <typename E, bool kInterleaved>
cudaError_t launch_rotary(const RotArgs& a, int v, dim3 grid, size_t smem, cudaStream_t st) {
  switch (v) {
    case 16:
      if constexpr (sizeof(E) == 2)
        return sl::launch(rotary_kernel<E, 16, kInterleaved>, grid, dim3(kRotThreads), smem, st, a);
      return cudaErrorInvalidValue;
    case 8: return sl::launch(rotary_kernel<E, 8, kInterleaved>, grid, dim3(kRotThreads), smem, st, a);
    case 4: return sl::launch(rotary_kernel<E, 4, kInterleaved>, grid, dim3(kRotThreads), smem, st, a);
    case 2: return sl::launch(rotary_kernel<E, 2, kInterleaved>, grid, dim3(kRotThreads), smem, st, a);
    default: return sl::launch(rotary_kernel<E, 1, kInterleaved>, grid, dim3(kRotThreads), smem, st, a);
  }
}

}  // namespace

extern "C" int sl_plan_kv_blocks(const int32_t* context_lens, const int32_t* new_lens, int B,
                                 int block_size, int32_t* block_table, int64_t ld_table,
                                 int table_width, const int32_t* free_blocks, int num_free_slots,
                                 const int64_t* free_range, int64_t* free_range_out, int64_t T,
                                 int64_t Tk, int32_t* cu_new, int32_t* cu_total,
                                 int64_t* positions, int64_t* slots, int64_t* kv_slots,
                                 int32_t* status, sl_stream_t stream) {
  if (B <= 0 || block_size <= 0 || table_width <= 0 || ld_table < table_width ||
      T < 0 || Tk < 0 || (Tk > 0 && !kv_slots))
    return SL_ERR_INVALID;
  const bool ring = free_blocks || free_range || free_range_out;
  if (ring && num_free_slots <= 0) return SL_ERR_INVALID;
  if (B > kPlanMaxRequests) return SL_ERR_UNSUPPORTED;
  if (!context_lens || !new_lens || !block_table ||
      (ring && (!free_blocks || !free_range || !free_range_out)) || !cu_new || !cu_total || !status || (T > 0 && (!positions || !slots)))
    return SL_ERR_INVALID;
  int shift = -1;
  if ((block_size & (block_size - 1)) == 0)
    for (shift = 0; (1 << shift) < block_size;) ++shift;
  PlanArgs a = {context_lens, new_lens, B, block_size, shift, table_width, num_free_slots, T, Tk,
                block_table, ld_table, free_blocks, free_range, free_range_out, cu_new, cu_total,
                positions, slots, Tk > 0 ? kv_slots : nullptr, status, 1};
  // Warps for a turn of the rows, up to 32 per SM. In small CTAs a scan has fewer
  // warps to wait for, in large ones fewer CTAs repeat it and there are more lanes
  // for it (us with 256, 512, 1024 threads): 8 requests 3.5, 3.7, 4.3; 256 of 64
  // rows 4.8, 5.2, 6.7; 1024 of 64 rows 7.5, 6.6, 7.4; 1024 of 2.2 million rows
  // together, several turns a warp, 20.6, 17.9, 16.1.
  const int64_t rows = T + Tk;
  const int sms = sl_device_sm_count();
  if (sms <= 0) return SL_ERR_CUDA;
  const int threads = rows > static_cast<int64_t>(sms) * 32 * kPlanChunk ? kPlanThreads
                      : B <= 256                                         ? 256
                                                                         : 512;
  const int64_t per_cta = kPlanChunk * (threads / 32);
  const int64_t most = static_cast<int64_t>(sms) * (kPlanThreads / threads);
  int64_t grid = (rows + per_cta - 1) / per_cta;
  grid = grid < 1 ? 1 : (grid > most ? most : grid);
  const bool in_place = ring && free_range_out == free_range;
  a.write_range = !(in_place && grid > 1);
  const size_t smem = sizeof(int) * (4 * static_cast<size_t>(B) + 2);
  static std::atomic<uint64_t> smem_set{0};
  if (smem > 40 * 1024)
    SL_CUDA_TRY(sl::ensure_smem_limit(plan_kv_blocks_kernel,
                                      sizeof(int) * (4 * kPlanMaxRequests + 2), smem_set));
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  SL_CUDA_TRY(sl::launch(plan_kv_blocks_kernel, dim3(static_cast<unsigned>(grid)),
                         dim3(threads), smem, st, a));
  if (!a.write_range)
    SL_CUDA_TRY(sl::launch(plan_range_kernel, dim3(1), dim3(1), 0, st, free_range_out,
                           static_cast<const int32_t*>(status)));
  return SL_OK;
}

extern "C" int sl_rotary(const int64_t* positions, const double* turns, int T, int rot,
                         int interleaved, float factor, int dtype, const sl_rotary_part* q,
                         const sl_rotary_part* k, sl_stream_t stream) {
  if (T < 0 || rot <= 0 || rot % 2 || !q || dtype < SL_DTYPE_BF16 || dtype > SL_DTYPE_FP32)
    return SL_ERR_INVALID;
  // (rows rounded up to a CTA's, of 32 at most, are still counted in 32 bits)
  if (rot > 2 * kRotMaxPairs || T > 0x7fffffff - 64) return SL_ERR_UNSUPPORTED;
  const sl_rotary_part none = {};
  const sl_rotary_part* parts[2] = {q, k ? k : &none};
  if (q->heads <= 0) return SL_ERR_INVALID;
  for (const sl_rotary_part* p : parts) {
    if (p->heads < 0) return SL_ERR_INVALID;
    if (p->heads == 0) continue;
    if (p->dim < rot || p->offset < 0 || p->offset > p->dim - rot) return SL_ERR_INVALID;
    if (T > 0 && (!p->x || !p->y)) return SL_ERR_INVALID;
    // (the unit index times the units of a head stays below 2^32)
    if (p->dim > 4096 || static_cast<int64_t>(p->heads) * p->dim >= (1 << 20))
      return SL_ERR_UNSUPPORTED;
  }
  if (T == 0) return SL_OK;
  if (!positions || !turns) return SL_ERR_INVALID;
  const int size = dtype == SL_DTYPE_FP32 ? 4 : 2;
  // the widest unit that divides every size, stride and address
  auto fits = [&](int v) {
    if (rot % (2 * v)) return false;
    for (const sl_rotary_part* p : parts) {
      if (p->heads == 0) continue;
      const int64_t all = static_cast<int64_t>(p->dim) | p->offset | p->x_token | p->x_head |
                          p->y_token | p->y_head;
      if (all % v || (reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->y)) %
                         static_cast<uintptr_t>(v * size))
        return false;
    }
    return true;
  };
  int v = 32 / size;
  while (v > 1 && !fits(v)) v >>= 1;
  RotArgs a = {};
  a.positions = positions;
  a.turns = turns;
  a.factor = factor;
  a.T = T;
  a.rot = rot;
  a.rot_units = rot / 2 / v;
  int items = 0;
  for (int i = 0; i < 2; ++i) {
    const sl_rotary_part* p = parts[i];
    RotTensor& t = a.t[i];
    t.units = 1;
    t.units_mul = 0;
    if (p->heads == 0) continue;
    const bool in_place = p->x == p->y && p->x_token == p->y_token && p->x_head == p->y_head;
    t.x = p->x;
    t.y = p->y;
    t.xs = p->x_token;
    t.xh = p->x_head;
    t.ys = p->y_token;
    t.yh = p->y_head;
    t.heads = p->heads;
    t.offset = p->offset;
    // in place the columns that are not rotated are left alone
    t.copied = in_place ? 0 : p->dim - rot;
    t.units = a.rot_units + (t.copied / v + 1) / 2;
    t.units_mul = t.units == 1 ? 0 : static_cast<uint32_t>(((1ull << 32) + t.units - 1) / t.units);
    items += t.heads * t.units;
  }
  // tokens per CTA: about four units per thread, so that the angles' sines
  // and cosines and the launch are spread over several rows; their table takes
  // 16 KB at most, for 8 CTAs per SM
  int per = 4 * kRotThreads / items;
  per = per < 1 ? 1 : (per > 32 ? 32 : per);
  const int sms = sl_device_sm_count();
  if (sms <= 0) return SL_ERR_CUDA;
  while (per > 1 && ((T + per - 1) / per < 4 * sms || per * rot * 4 > 16 * 1024)) per >>= 1;
  a.per_cta = per;
  a.inv_items = 1.f / static_cast<float>(items);
  const dim3 grid((T + per - 1) / per);
  const size_t smem = static_cast<size_t>(per) * (rot / 2) * sizeof(float2);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == SL_DTYPE_BF16)
    e = interleaved ? launch_rotary<__nv_bfloat16, true>(a, v, grid, smem, st)
                    : launch_rotary<__nv_bfloat16, false>(a, v, grid, smem, st);
  else if (dtype == SL_DTYPE_FP16)
    e = interleaved ? launch_rotary<__half, true>(a, v, grid, smem, st)
                    : launch_rotary<__half, false>(a, v, grid, smem, st);
  else
    e = interleaved ? launch_rotary<float, true>(a, v, grid, smem, st)
                    : launch_rotary<float, false>(a, v, grid, smem, st);
  SL_CUDA_TRY(e);
  return SL_OK;
}
