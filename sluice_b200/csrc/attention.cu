// Causal attention over packed sequences with grouped heads, on the fifth
// generation tensor cores.
//
//   out_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i . k_j - m_i),
//   j <= i + keys - queries
//
// One pass over the keys with a running maximum m and a running sum, both in 32
// bits; the weights are rounded once, to the inputs' type, as the second
// product's operand. An item is 2 x 128 rows of one sequence and key head; its
// rows are (token, head of the group) pairs, so a single token of a wide group
// fills rows that would otherwise be empty, and a key tile is read once for all
// heads of its group. Per item and 128-key tile: S = Q K^T (128 x 128 per 128
// rows, fp32, in TMEM), the softmax warpgroup of those rows reads a row per
// thread, writes the weights P over S, and O += P V takes P from TMEM.
//
// Roles (12 warps): 0-3 and 4-7 softmax of the two halves (a row per thread)
// and their output; 8 and 11 issue the MMAs of a half each; 9 the tile loads
// (TMA); 10 publishes the stretches of work one ahead and cleans the value tiles
// that hold keys which some row may not see.
//
// Shared memory: the item's queries (2 x 128 rows) and a ring of 16 KB slots
// that the key and value tiles pass through: 64 columns of 128 keys, or 64
// value rows of 128 columns.
//
// What bounds it. A tile of both halves is 2048 cycles of MMAs (dim 128; 2560 at
// 192) and 2048 of exponentials (16 a cycle and SM). One half's chain - scores,
// maximum, exponentials, hand-over, both products - is longer than either, so
// the halves run half a step apart: their warps take turns at the exponentials
// (without the turns both wait for the special-function units, then both for the
// tensor core: 4096 tokens on 16 heads of 192 / 128 took 95 us instead of 74).
// Then the hand-overs count: named barriers instead of mbarriers between warps,
// waits without a suspend hint or a vote (82 -> 74 us), the maximum taken outside
// the turn (16384 tokens on 32 / 4 heads of 128: 1.93 -> 1.77 ms). Now, device time:
//   4096 tokens, 16 heads of 192 / 128        73 us, 1180 TFLOP/s, 0.72 of cuBLAS's burst
//   16384 tokens, 32 / 4 heads of 128       1.88 ms, 1172 TFLOP/s, 0.86 of cuBLAS's
//                                             sustained rate (the power cap; 1.64 ms before)
//   8 single tokens over 60 000 keys, 32 / 4  34 us, 19 of them the bytes; 8 until the first
//                                             scores are there, 5 for the join
// Measured and not kept: part of the exponentials as a cubic on the FMA pipes
// (73.5 us with a quarter against 72.5), 16 softmax warps with a row in two
// threads (90 against 82), the turn passed on after half the weights (80
// against 74), the scores waited for within the turn (85 against 82).
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"

namespace {

constexpr int kThreads = 384;
constexpr int kTile = 128;           // rows of a half and keys of a tile
constexpr int kSlotBytes = 16384;
constexpr int kCoarse = 256;         // entries of the work table
constexpr int kBars = 16;            // barriers of tiles in flight; even ones keys, odd ones values
// How far (in powers of 2) a row's maximum may lag behind its scores, and the
// power of 2 that its weight is. bf16 weights have the exponents of the 32-bit
// sums: 2^16 keys, each at the lag's end, have a sum of weights of at most one, so
// that no sum of weighted values passes the largest value (weights below 2^-86 of
// the maximum's become zero). fp16 ones end at 2^16 and, below 2^-14, lose bits: of
// weights of 2^-21 of the maximum's and less, 2^-33 of its, so that 2^21 keys lose
// half an output's rounding at most. A smaller lag moves the maximum more often:
// bf16, 16384 tokens on 8 / 2 heads of 128, scores that spread by 1, 3 and 6, 409,
// 413 and 415 us; with a lag of 8 410, 443 and 492, of 32 410, 412 and 410. fp16,
// 8192 tokens on 16 / 4 heads, scores that spread by 3, 245; with 4, which would
// keep weights 2^4 smaller, 276, with 12 228.
constexpr float kLagBf16 = 24.f, kLagF16 = 8.f;
constexpr float kTopBf16 = -40.f, kTopF16 = 7.f;
// registers a thread: 168 at launch, then shared out between the softmax warps
// and the others (256 x 216 + 128 x 72 = 384 x 168)
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
constexpr int kReaders = 11;          // warps that follow the stretches
constexpr int kSegs = 4;              // stretches looked up ahead
constexpr int kItemUnits = 3;         // what starting and ending an item costs, in key tiles
constexpr int kMarks = 16;           // items that the value guards may be ahead by

// What the join needs to know of a CTA's first stretch: the item it is a later
// part of (unit0 < 0: of none).
struct Later {
  int unit0, q0, q_len, k_len, tok, head, pad[2];
};

// x / d of 0 <= x < 2^31 by a multiplication: mul = ceil(2^(31 + shift) / d),
// 2^shift >= d (a division by a number that is not known when compiling is a
// long subroutine, and the lookups of a stretch are all divisions).
struct Divisor {
  uint32_t mul;
  int shift, d;
};
__device__ __forceinline__ int quotient(const Divisor& v, int x) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(x)) * v.mul) >> (31 + v.shift));
}

struct Params {
  CUtensorMap q, k, v, ks;
  void* out;
  int64_t out_token, out_head;
  const int32_t* cu_q;
  const int32_t* cu_k;
  // inputs as they are, for the rare repair of a column
  const void *vraw, *qraw, *kraw, *ksraw;
  int64_t v_token, v_head, q_token, q_head, k_token, k_head, ks_token;
  int B, Tq, Tk, heads, kv_heads, group, half_tokens;  // tokens of a half: 128 / group
  int shared;                        // the last 64 key columns come from ks
  int wide;                          // the output's rows are 32-byte aligned: stores of 32 bytes
                                     // (2048 tokens, 16 heads of 128: 38.8 us, of 16 bytes 40.8)
  int grid;                          // CTAs
  Divisor by_tokens, by_heads, by_grid;  // tokens of an item, key heads, CTAs
  int split;                         // 1: equal shares of all key tiles per CTA
  int rows_cap;                      // rows of a partial result
  float scale_log2;                  // scale / ln 2
  float lag;                         // how far the maximum may lag behind, in scores
  float* part;                       // [2 * grid][rows_cap][v_dim]
  float2* part_ml;                   // [2 * grid][rows_cap] (maximum, sum)
  Later* later;                      // [grid]
  int32_t* status;                   // of this call
  int32_t* failed;                   // of many calls: only ever raised (nullptr: not asked for)
};

// ------------------------------------------------------------------ helpers
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(sl::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(sl::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// Shared-memory matrix descriptors of 128-byte swizzled tiles: 8-row groups
// 1024 bytes apart (high word, with the version and the swizzle); the low word
// is the address / 16 and the step between 64-column groups / 16. An operand
// whose rows hold the reduction index's values (queries, keys) has one group
// per row; one whose rows are the reduction index (values: a row per key) has
// the next 64 columns a group of rows further.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kKMajorLo = 1u << 16;
template <int kRows>
constexpr uint32_t kRowMajorLo = static_cast<uint32_t>(kRows * 128 >> 4) << 16;

// D (+)= A B, both from shared memory.
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi)
      : "memory");
}
// D (+)= A B, A from TMEM (the weights).
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi)
      : "memory");
}
__host__ __device__ constexpr uint32_t idesc_f16(bool bf16, int N, bool b_rows) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_rows ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_fence_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}
// Eight columns of this thread's row times f.
__device__ __forceinline__ void tmem_scale8(uint32_t taddr, float f) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(
                   taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
               "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 32 bytes to a 32-byte aligned address
__device__ __forceinline__ void store32(void* to, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// the largest of three; NaN if any is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t d;
  if constexpr (kBf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

__device__ __forceinline__ void report(const Params& p, int status) {
  atomicMax(p.status, status);
  if (p.failed != nullptr) atomicMax(p.failed, status);
}

// A role's outlook: once a bounded wait has run out, it waits for nothing more
// and issues nothing more, but walks its work to the end, so that the named
// barriers, which have no limit of their own, still meet all their warps.
struct Outlook {
  bool ok = true;
  // A bounded wait of a whole warp: its lanes run the same instructions on the
  // same word, so they agree on the outcome. (Without the suspend-time hint of
  // sl::mbar_wait: a signal takes 108 cycles instead of 137, a wait that is
  // over already 14 instead of 49.)
  __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
    if (ok && !try_wait(bar, parity)) {
      const uint64_t t0 = sl::globaltimer();
      for (uint32_t i = 1; ok; ++i) {
        if (try_wait(bar, parity)) break;
        if ((i & 15u) == 0 && sl::globaltimer() - t0 > sl::kWaitLimitNs) ok = false;
      }
    }
    __syncwarp();
    return ok;
  }
  static __device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(sl::smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
  }
};
// Named barriers (a signal between warps takes a tenth of an mbarrier's): `n`
// threads in all, those that wait and those that only arrive.
__device__ __forceinline__ void bar_wait(int id, int n) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int n) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory");
}
constexpr int kBarTurn = 1;     // + 4 * half + quad: this half's turn; 64 threads
constexpr int kBarWeights = 9;  // + 2 * half + part: weights are there; 160 threads
constexpr int kBarTwin = 13;    // half 1's result is there; 256 threads

// --------------------------------------------------------------------- work
// One stretch of an item's key tiles: [j0, j1) of n.
struct Seg {
  int seq, tile, head;
  int q0, q_len, k0, k_len;   // the sequence's rows, clamped to the tensors
  int tok;                    // first token of the item
  int n, j0, j1;              // key tiles of the item, and this stretch
  int nh[2];                  // key tiles that each half's last row reaches
  int lim0;                   // keys that the item's first row sees
};

// Where an item's rows fill one half only, both halves take them, each every
// other key tile of the stretch, and their results are joined at its end (short
// prompts with such tails 38 -> 36 us; from two tiles on, so that each has one).
__device__ __forceinline__ bool is_twin(const Seg& g) { return g.nh[1] == 0 && g.j1 - g.j0 >= 2; }

struct Seq {
  int q0, q_len, k0, k_len;
};

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return max(lo, min(v, hi)); }

__device__ __forceinline__ Seq load_seq(const Params& p, int s) {
  Seq r;
  r.q0 = clampi(p.cu_q[s], 0, p.Tq);
  r.q_len = clampi(p.cu_q[s + 1], r.q0, p.Tq) - r.q0;
  r.k0 = clampi(p.cu_k[s], 0, p.Tk);
  r.k_len = clampi(p.cu_k[s + 1], r.k0, p.Tk) - r.k0;
  return r;
}
// keys that token `tok` of a sequence sees
__device__ __forceinline__ int seen(const Seq& s, int tok) {
  return clampi(tok + 1 + s.k_len - s.q_len, 0, s.k_len);
}
__device__ __forceinline__ int tiles_of(const Params& p, const Seq& s) {
  return quotient(p.by_tokens, s.q_len) + (quotient(p.by_tokens, s.q_len) * p.by_tokens.d < s.q_len);
}
// key tiles of item `t`
__device__ __forceinline__ int reach(const Params& p, const Seq& s, int t) {
  const int last = min(s.q_len, (t + 1) * 2 * p.half_tokens) - 1;
  return (seen(s, last) + kTile - 1) / kTile;
}
__device__ __forceinline__ int64_t work_of(const Params& p, const Seq& s) {
  const int nt = tiles_of(p, s);
  if (!p.split) return nt;
  int64_t w = 0;
  for (int t = 0; t < nt; ++t) w += kItemUnits + reach(p, s, t);
  return w;
}

// cum[i]: work of the sequences before the i-th run of `per` ones (in items,
// or in key tiles where items are split); all threads take part.
__device__ __forceinline__ void build_table(const Params& p, int* cum, int* warp_sum, int per) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t w = 0;
  if (tid < kCoarse)
    for (int s = tid * per; s < min(p.B, (tid + 1) * per); ++s) w += work_of(p, load_seq(p, s));
  int v = static_cast<int>(min(w, static_cast<int64_t>(1 << 22)));
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (tid < kCoarse && lane == 31) warp_sum[warp] = v;
  __syncthreads();
  if (tid < kCoarse) {
    for (int i = 0; i < warp; ++i) v += warp_sum[i];
    cum[tid + 1] = v;
    if (tid == 0) cum[0] = 0;
  }
  __syncthreads();
}

// The sequence that unit u falls in, and u's place in it (warp-uniform).
__device__ __forceinline__ Seq find_seq(const Params& p, const int* cum, int per, int u, int& seq,
                                        int& rest) {
  const int lane = threadIdx.x & 31;
  int c = 0;
#pragma unroll
  for (int i = 0; i < kCoarse / 32; ++i) c += cum[lane * (kCoarse / 32) + i + 1] <= u;
  const int run = __reduce_add_sync(0xffffffffu, c);
  rest = u - cum[run];
  const int end = min(p.B, (run + 1) * per);
  seq = run * per;
  if (per > 1) {
    for (int s0 = seq;; s0 += 32) {
      const int s = s0 + lane;
      const int own = s < end ? static_cast<int>(work_of(p, load_seq(p, s))) : 0;
      int v = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, v > rest);
      if (hit || s0 + 32 >= end) {
        const int l = hit ? __ffs(hit) - 1 : 0;
        seq = s0 + l;
        rest -= __shfl_sync(0xffffffffu, v - own, l);
        break;
      }
      rest -= __shfl_sync(0xffffffffu, v, 31);
    }
  }
  return load_seq(p, seq);
}

__device__ __forceinline__ void fill_seg(const Params& p, const Seq& s, Seg& g) {
  g.q0 = s.q0;
  g.q_len = s.q_len;
  g.k0 = s.k0;
  g.k_len = s.k_len;
  g.tok = g.tile * 2 * p.half_tokens;
  g.lim0 = seen(s, g.tok);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int first = g.tok + h * p.half_tokens;
    const int last = min(s.q_len, first + p.half_tokens) - 1;
    g.nh[h] = first < s.q_len ? (seen(s, last) + kTile - 1) / kTile : 0;
  }
  g.n = max(g.nh[0], g.nh[1]);
}

// The parts of a stretch that steer the issuing warps, as values that the
// compiler knows to be the same in all lanes.
__device__ __forceinline__ void uniform(Seg& g) {
  constexpr unsigned kAll = 0xffffffffu;
  g.head = __shfl_sync(kAll, g.head, 0);
  g.q0 = __shfl_sync(kAll, g.q0, 0);
  g.k0 = __shfl_sync(kAll, g.k0, 0);
  g.k_len = __shfl_sync(kAll, g.k_len, 0);
  g.tok = __shfl_sync(kAll, g.tok, 0);
  g.j0 = __shfl_sync(kAll, g.j0, 0);
  g.j1 = __shfl_sync(kAll, g.j1, 0);
  g.nh[0] = __shfl_sync(kAll, g.nh[0], 0);
  g.nh[1] = __shfl_sync(kAll, g.nh[1], 0);
  g.lim0 = __shfl_sync(kAll, g.lim0, 0);
}

// How many of a sequence's nt items reach x > 0 key tiles or more (they are its
// last ones: what an item reaches grows with its place).
__device__ __forceinline__ int items_from(const Params& p, const Seq& s, int nt, int x) {
  const int need = (x - 1) * kTile + 1;  // keys that the item's last row sees, at least
  if (nt == 0 || s.k_len < need) return 0;
  const int m = need - (s.k_len - s.q_len);  // ... which is so from this row on
  const int t = m <= p.by_tokens.d ? 0 : quotient(p.by_tokens, m + p.by_tokens.d - 1) - 1;
  return nt - min(t, nt - 1);
}

// The ord-th item, as (sequence, place), in the order of the key tiles that
// items reach, most first; of up to 32 sequences, a lane each.
__device__ __noinline__ int2 pick_item(const Params& p, int ord) {
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  Seq mine = {0, 0, 0, 0};
  if (lane < p.B) mine = load_seq(p, lane);
  // the largest x that more than ord items reach; from: this lane's that do,
  // more: those that reach further
  const int nt = tiles_of(p, mine);
  int x = 0, from = nt, more = 0, past = 0;  // past: all lanes' that reach further
  int hi = __reduce_max_sync(kAll, (mine.k_len + kTile - 1) / kTile) + 1;
  while (hi - x > 1) {
    const int mid = (x + hi) >> 1;
    const int mine_from = items_from(p, mine, nt, mid);
    const int n = __reduce_add_sync(kAll, mine_from);
    if (n > ord) {
      x = mid;
      from = mine_from;
    } else {
      hi = mid;
      past = n;
      more = mine_from;
    }
  }
  const int own = from - more;
  int v = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(kAll, v, o);
    if (lane >= o) v += u;
  }
  const int rest = ord - past;
  const int l = max(0, __ffs(__ballot_sync(kAll, v > rest)) - 1);
  return make_int2(l, __shfl_sync(kAll, nt - from + rest - (v - own), l));
}

// Walks a CTA's share of the work.
//   whole items: the longest first (of up to 32 sequences, a lane each; of more,
//   sequence after sequence), dealt out in turns that go back and forth (16
//   prompts of 1 to 1024 tokens: 28 us, sequence after sequence 37);
//   split: an equal run of key tiles, item after item.
struct Walk {
  int total, at, end, round, unit0;  // unit0: the first unit of the last stretch's item
  bool sorted;

  __device__ void start(const Params& p, const int* cum) {
    total = units(p, cum);
    round = 0;
    // (one sequence is in order already, and the order does not matter where no
    // CTA takes a second item)
    sorted = !p.split && p.B > 1 && p.B <= 32 && total > p.grid;
    if (p.split) {
      at = share(p, total, blockIdx.x);
      end = share(p, total, blockIdx.x + 1);
    }
  }
  __device__ static int units(const Params& p, const int* cum) {
    return static_cast<int>(min(static_cast<int64_t>(cum[kCoarse]) * p.kv_heads,
                                static_cast<int64_t>(1 << 30)));
  }
  // where CTA c's share begins: equal ones, the first with one unit more
  __device__ static int share(const Params& p, int total, int c) {
    const int each = quotient(p.by_grid, total);
    return each * c + min(c, total - each * p.grid);
  }
  __device__ bool next(const Params& p, const int* cum, int per, Seg& g) {
    if (!p.split) {
      const int G = p.grid;
      const int c = blockIdx.x;
      const int i = round * G + ((round & 1) ? G - 1 - c : c);
      if (i >= total) return false;
      ++round;
      const int ord = quotient(p.by_heads, i);
      g.head = i - ord * p.kv_heads;
      Seq s;
      if (sorted) {
        const int2 at = pick_item(p, ord);
        g.seq = at.x;
        g.tile = at.y;
        s = load_seq(p, g.seq);
      } else {
        int rest;
        s = find_seq(p, cum, per, ord, g.seq, rest);
        g.tile = tiles_of(p, s) - 1 - rest;
      }
      fill_seg(p, s, g);
      g.j0 = 0;
      g.j1 = g.n;
      return true;
    }
    // (a share may begin or end within an item's first units, which are no key
    // tiles: that stretch is empty, and skipped unless it is the whole item)
    while (at < end) {
      int j, n;
      locate(p, cum, per, at, g, j, n);
      unit0 = at - j;
      const int to = min(n, j + end - at);
      at += to - j;
      g.j0 = max(0, j - kItemUnits);
      g.j1 = max(0, to - kItemUnits);
      if (g.j0 < g.j1 || (g.n == 0 && to == n)) return true;
    }
    return false;
  }
  // The item that unit u falls in, u its j-th of n units: kItemUnits for the
  // item itself, then one for each key tile.
  __device__ static void locate(const Params& p, const int* cum, int per, int u, Seg& g, int& j,
                                int& n) {
    const int lane = threadIdx.x & 31;
    // units of a sequence count all heads: tile after tile, head after head
    int rest;
    const int ord = quotient(p.by_heads, u);
    const Seq s = find_seq(p, cum, per, ord, g.seq, rest);
    int r = rest * p.kv_heads + u - ord * p.kv_heads;
    const int nt = tiles_of(p, s);
    for (int t0 = 0;; t0 += 32) {
      const int t = t0 + lane;
      const int own = t < nt ? (kItemUnits + reach(p, s, t)) * p.kv_heads : 0;
      int v = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, v > r);
      if (hit || t0 + 32 >= nt) {
        const int l = hit ? __ffs(hit) - 1 : 0;
        g.tile = t0 + l;
        r -= __shfl_sync(0xffffffffu, v - own, l);
        break;
      }
      r -= __shfl_sync(0xffffffffu, v, 31);
    }
    fill_seg(p, s, g);
    n = kItemUnits + g.n;
    // r / n (the estimate is off by one at most: r < 2^22)
    g.head = static_cast<int>(__fdividef(static_cast<float>(r), static_cast<float>(n)));
    j = r - g.head * n;
    if (j < 0) {
      --g.head;
      j += n;
    } else if (j >= n) {
      ++g.head;
      j -= n;
    }
  }
};

// ------------------------------------------------------------------- kernel
template <int kDim, int kVDim>
struct Cfg {
  static constexpr int kChunks = kDim / 64;                  // 64-column slots of a key tile
  static constexpr int kVSlots = kVDim / 64;                 // slots of a value tile
  static constexpr int kVRows = kTile / kVSlots;             // keys of a value slot
  static constexpr int kQBytes = 2 * kChunks * kSlotBytes;
  static constexpr int kSlots = (14 * kSlotBytes - kQBytes) / kSlotBytes;  // 8, 10, 12
  static constexpr int kBufBytes = kQBytes + kSlots * kSlotBytes;          // 224 KB
};

struct Sync {
  uint64_t full[kBars], empty[kBars], clean[kBars];
  uint64_t q_full[2], q_empty[2], s_full[2], pv_done[2], o_free[2], drain[2];
  uint64_t seg_full[kSegs], seg_empty[kSegs];
  Seg seg[kSegs];
  uint32_t tmem;
  float2 twin[kTile];  // half 1's (maximum, sum) of each row
  int mark[kMarks];
  int warp_sum[kCoarse / 32];
  int cum[kCoarse + 1];
};
constexpr int kSmemBytes = 14 * kSlotBytes + static_cast<int>(sizeof(Sync));
static_assert(kSmemBytes <= 232448, "shared memory of a CTA");

// A role's place in the sequence of tiles (keys, values, keys, ...): the
// tile's number, which names its barriers and their parity, and its first slot.
// At most kSlots tiles are in flight, fewer than there are barriers, and each is
// let go by all that wait for it before its slots are filled again.
struct Tiles {
  uint32_t n = 0;
  int slot = 0;
  __device__ __forceinline__ int bar() const { return n % kBars; }
  __device__ __forceinline__ uint32_t phase() const { return (n / kBars) & 1; }
  template <int N>
  __device__ __forceinline__ int place(int i) const {
    return slot + i < N ? slot + i : slot + i - N;
  }
  template <int N>
  __device__ __forceinline__ void step(int slots) {
    slot = place<N>(slots);
    ++n;
  }
};

// Rows [lo, rows) of a value group (128-byte rows in shared memory, any
// swizzle): those from hi on are zeroed, and values that are not finite in
// the others. Whether there were any. One warp; the look is cheap and its
// loads run ahead (an exponent of all ones carries into the sign's place when
// one is added to it), the repair is rare.
template <bool kBf16>
__device__ __forceinline__ bool clean_rows(uint8_t* base, int lo, int hi, int rows, int lane) {
  constexpr uint32_t kExp = kBf16 ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t kOne = kBf16 ? 0x00800080u : 0x04000400u;
  for (int x = max(lo, hi) * 8 + lane; x < rows * 8; x += 32)
    *reinterpret_cast<uint4*>(base + x * 16) = make_uint4(0, 0, 0, 0);
  bool found = false;
  // 32 rows a turn, eight loads of a lane in flight
  for (int x0 = lo * 8; x0 < hi * 8; x0 += 256) {
    uint4 w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int x = x0 + 32 * i + lane;
      // (past the last row: row lo once more)
      w[i] = *reinterpret_cast<const uint4*>(base + (x < hi * 8 ? x : lo * 8 + (lane & 7)) * 16);
    }
    uint32_t carry = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      carry |= ((w[i].x & kExp) + kOne) | ((w[i].y & kExp) + kOne) | ((w[i].z & kExp) + kOne) |
               ((w[i].w & kExp) + kOne);
    if (!__any_sync(0xffffffffu, carry & 0x80008000u)) continue;
    found = true;
    for (int x = x0 + lane; x < min(hi * 8, x0 + 256); x += 32) {
      uint32_t* e = reinterpret_cast<uint32_t*>(base + x * 16);
      for (int k = 0; k < 4; ++k) {
        uint32_t v = e[k];
        if ((v & kExp & 0xffffu) == (kExp & 0xffffu)) v &= 0xffff0000u;
        if ((v & kExp & 0xffff0000u) == (kExp & 0xffff0000u)) v &= 0xffffu;
        e[k] = v;
      }
    }
  }
  return found;
}

// Whether the weight of a key is zero as the second product takes it, against a
// row's maximum m. One thread.
template <int kDim, bool kBf16>
__device__ __noinline__ bool no_weight(const Params& p, float m, int row, int head, int key_row,
                                       int key_head) {
  auto f = [](uint16_t b) {
    return kBf16 ? __uint_as_float(static_cast<uint32_t>(b) << 16)
                 : __half2float(__ushort_as_half(b));
  };
  const uint16_t* q = static_cast<const uint16_t*>(p.qraw) + row * p.q_token + head * p.q_head;
  const uint16_t* k = static_cast<const uint16_t*>(p.kraw) + key_row * p.k_token +
      key_head * p.k_head;
  const int own = p.shared ? kDim - 64 : kDim;
  float s = 0.f;
  for (int c = 0; c < own; ++c) s = fmaf(f(q[c]), f(k[c]), s);
  const uint16_t* ks = static_cast<const uint16_t*>(p.ksraw) + key_row * p.ks_token;
  for (int c = own; c < kDim; ++c) s = fmaf(f(q[c]), f(ks[c - own]), s);
  const float top = kBf16 ? kTopBf16 : kTopF16;
  const float w = m == -INFINITY ? 0.f
                                 : ex2(fmaf(s, p.scale_log2, __fadd_rn(__fmul_rn(-m, p.scale_log2), top)));
  return pack2<kBf16>(w, w) == 0;
}

template <int kDim, int kVDim, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1) attention_kernel(
    const __grid_constant__ Params p) {
  using C = Cfg<kDim, kVDim>;
  extern __shared__ __align__(1024) uint8_t buf[];
  uint8_t* ring = buf + C::kQBytes;
  Sync& sy = *reinterpret_cast<Sync*>(buf + C::kBufBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int per = (p.B + kCoarse - 1) / kCoarse;

  if (sl::smem_u32(buf) & 1023) {
    // (the swizzled tiles want it; there is no static shared memory before it)
    if (tid == 0) {
      *p.status = SL_OK;
      report(p, SL_ERR_UNSUPPORTED);
    }
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < kBars; ++i) {
      sl::mbar_init(&sy.full[i], 1);
      // both halves' MMAs, and of a value tile the guard, which may be late: it
      // tells the uses of a barrier apart by their parity, so none may pass it by
      sl::mbar_init(&sy.empty[i], i % 2 ? 3 : 2);
      sl::mbar_init(&sy.clean[i], 1);
    }
    for (int h = 0; h < 2; ++h) {
      sl::mbar_init(&sy.q_full[h], 1);
      sl::mbar_init(&sy.q_empty[h], 1);
      sl::mbar_init(&sy.s_full[h], 1);
      sl::mbar_init(&sy.pv_done[h], 1);
      sl::mbar_init(&sy.o_free[h], 4);
      sl::mbar_init(&sy.drain[h], 1);
    }
    for (int i = 0; i < kMarks; ++i) sy.mark[i] = -1;
    for (int i = 0; i < kSegs; ++i) {
      sl::mbar_init(&sy.seg_full[i], 1);
      sl::mbar_init(&sy.seg_empty[i], kReaders);
    }
    sl::fence_barrier_init();
  }
  if (warp == 8) sl::tmem_alloc(&sy.tmem, 512);
  if (tid == kThreads - 1) {
    sl::tma_prefetch_desc(&p.q);
    sl::tma_prefetch_desc(&p.k);
    sl::tma_prefetch_desc(&p.v);
  }
  sl::pdl_wait();
  sl::pdl_trigger();
  if (blockIdx.x == 0 && tid == 0) *p.status = SL_OK;
  build_table(p, sy.cum, sy.warp_sum, per);  // (its barriers publish the set-up above)
  sl::tc_fence_before();
  __syncthreads();
  sl::tc_fence_after();
  const uint32_t tmem = sy.tmem;
  const uint32_t s_col[2] = {tmem, tmem + kTile};
  const uint32_t o_col[2] = {tmem + 2 * kTile, tmem + 2 * kTile + kVDim};
  Outlook out;
  // The stretches of this CTA's share, as the guard's warp publishes them, one
  // ahead of its own work: looking one up takes microseconds. (Waited for even
  // when something else has run out, so that all roles stop at the same one.)
  Seg g;
  int n_seg = 0;
  auto next_seg = [&]() -> bool {
    const int i = n_seg % kSegs;
    Outlook here;
    if (!here.wait(&sy.seg_full[i], (n_seg / kSegs) & 1)) return out.ok = false;
    g = sy.seg[i];
    ++n_seg;
    __syncwarp();
    if (lane == 0) sl::mbar_arrive(&sy.seg_empty[i]);
    return g.seq >= 0;
  };

  if (warp < 8) {
    // ---------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int h = warp >> 2;
    const int row = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // (warp mod 4) * 32 lanes
    const uint32_t s_at = s_col[h] + lanes, o_at = o_col[h] + lanes;
    const int token = row / p.group, in_group = row - token * p.group;
    const bool packed = token < p.half_tokens;
    int n_s = 0, n_item = 0;  // key tiles so far; items with keys so far
    // The warps of the two halves that share a scheduler take turns at the
    // exponentials, so that one half's run while the other's products do.
    const int quad = warp & 3;
    bool free_turn = h == 0;
    auto take_turn = [&]() {
      if (!free_turn) bar_wait(kBarTurn + 4 * h + quad, 64);
      free_turn = false;
    };
    auto pass_turn = [&]() {
      __syncwarp();
      bar_arrive(kBarTurn + 4 * (h ^ 1) + quad, 64);
    };
    while (next_seg()) {
      const bool twin = is_twin(g);
      const int first = g.tok + (twin ? 0 : h * p.half_tokens);
      const int j0 = twin ? g.j0 + h : g.j0, step = twin ? 2 : 1;
      const int j1 = twin ? g.j1 : min(g.j1, h ? g.nh[1] : g.nh[0]);
      const bool has = g.j0 < g.j1;
      const int mark = has ? n_item++ : -1;
      if (first >= g.q_len) {
        for (int j = g.j0; j < g.j1; ++j) {
          take_turn();
          pass_turn();
        }
        continue;
      }
      const int tok = first + token;
      const bool live = packed && tok < g.q_len;
      const int lim = live ? clampi(tok + 1 + g.k_len - g.q_len, 0, g.k_len) : 0;
      const int lim_first = clampi(first + 1 + g.k_len - g.q_len, 0, g.k_len);
      // base: -m in powers of 2, and the power that its own weight is
      float m = -INFINITY, l = 0.f, base = 0.f;
      constexpr float kTop = kBf16 ? kTopBf16 : kTopF16;
      for (int j = j0; j < j1; j += step) {
        out.wait(&sy.s_full[h], n_s & 1);
        sl::tc_fence_after();
        uint32_t r[kTile];
        auto s = [&](int c) { return __uint_as_float(r[c]); };
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_at + 32 * c, r + 32 * c);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_fence_ld(r + 32 * c);
        if ((j + 1) * kTile > lim_first) {
          const int left = lim - j * kTile;
#pragma unroll
          for (int c = 0; c < kTile; ++c)
            if (c >= left) r[c] = 0xff800000u;  // -inf
        }
        float top;
        {
          float t[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) t[i] = max3(s(32 * i), s(32 * i + 1), s(32 * i + 2));
#pragma unroll
          for (int c = 3; c < 31; c += 2)
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = max3(t[i], s(32 * i + c), s(32 * i + c + 1));
#pragma unroll
          for (int i = 0; i < 4; ++i) t[i] = max2(t[i], s(32 * i + 31));
          top = max2(max3(t[0], t[1], t[2]), t[3]);
        }
        // The weights are formed against a maximum that may lag behind this
        // tile's by a factor 2^kLag (the sums and the weights' type hold that);
        // only where it is beyond, or NaN, the rows move to it.
        const bool move = live && !(top <= m + p.lag);
        if (__any_sync(0xffffffffu, move)) {
          // a score of +inf leaves no finite weights: the row is NaN, as
          // inf - inf makes it
          if (top == INFINITY) top = __int_as_float(0x7fffffff);
          const float corr = move ? ex2((m - top) * p.scale_log2) : 1.f;
          if (move) m = top;
          // (two roundings: fused to one, the compiler's order of the loop takes
          // 77 us for 4096 tokens instead of 72)
          base = m == -INFINITY ? 0.f : __fadd_rn(__fmul_rn(-m, p.scale_log2), kTop);
          l *= corr;
          if (j > j0) {
            // the sums so far, once the products before this tile are in
            out.wait(&sy.pv_done[h], (n_s - 1) & 1);
            sl::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < kVDim / 8; ++c) tmem_scale8(o_at + 8 * c, corr);
          }
        }
        float2 sum = make_float2(0.f, 0.f);
        // Scores 2 c0 .. 2 c1 - 1 as weights, in place and packed.
        auto weights = [&](int c0, int c1) {
          const float2 sc = make_float2(p.scale_log2, p.scale_log2), bs = make_float2(base, base);
#pragma unroll
          for (int c = c0; c < c1; ++c) {
            float2 x = __ffma2_rn(make_float2(s(2 * c), s(2 * c + 1)), sc, bs);
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            sum = __fadd2_rn(sum, x);
            r[c] = pack2<kBf16>(x.x, x.y);
          }
        };
        // Handed over in halves: the product with the first 64 values runs
        // while the weights of the others are formed.
        auto hand_over = [&](int part) {
          tmem_wait_st();
          sl::tc_fence_before();
          __syncwarp();
          bar_arrive(kBarWeights + 2 * h + part, 160);
        };
        take_turn();
        weights(0, 32);
        tmem_st32(s_at, r);
        hand_over(0);
        // (the other half's first exponentials come in behind the last ones: 4096
        // tokens 72.1 us, the turn passed on after all of them 73.0)
        weights(32, 60);
        pass_turn();
        weights(60, 64);
        tmem_st32(s_at + 32, r + 32);
        hand_over(1);
        l += sum.x + sum.y;
        ++n_s;
      }
      // (the other half may have more tiles)
      const int spare = twin ? (g.j1 - g.j0) & h : g.j1 - max(g.j0, j1);
      for (int j = 0; j < spare; ++j) {
        take_turn();
        pass_turn();
      }
      // ------------------------------------------------------- output
      const bool whole = g.j0 == 0 && g.j1 == g.n;
      const int out_row = g.q0 + tok, out_head = g.head * p.group + in_group;
      const int prow = h * p.half_tokens * p.group + row;
      const int pslot = 2 * blockIdx.x + (g.j0 > 0 ? 0 : 1);
      float* part = p.part + (static_cast<int64_t>(pslot) * p.rows_cap + prow) * kVDim;
      const bool ran = j0 < j1;
      if (ran) {
        out.wait(&sy.pv_done[h], (n_s - 1) & 1);
        sl::tc_fence_after();
      }
      // twin: half 0 puts the two results together, row by row (the same TMEM
      // lanes, the other accumulator)
      float own = 1.f, others = 0.f;
      if (twin) {
        if (h == 1) {
          sy.twin[row] = make_float2(m, l);
          sl::tc_fence_before();
          __syncwarp();
          bar_arrive(kBarTwin, 256);
          continue;
        }
        bar_wait(kBarTwin, 256);
        sl::tc_fence_after();
        const float2 ml = sy.twin[row];
        const float top = max2(m, ml.x), to = top == -INFINITY ? 0.f : top;
        own = ex2((m - to) * p.scale_log2);
        others = ex2((ml.x - to) * p.scale_log2);
        m = top;
        l = l * own + ml.y * others;
      }
      if (!whole && live) p.part_ml[static_cast<int64_t>(pslot) * p.rows_cap + prow] =
          make_float2(m, l);
      const bool repair = has && sy.mark[mark % kMarks] == mark;
      // no key seen: zeros; only keys that score -inf: 0 / 0
      const float inv = lim == 0 ? 0.f : m == -INFINITY ? __int_as_float(0x7fffffff) : 1.f / l;
      uint16_t* dst = static_cast<uint16_t*>(p.out) +
          static_cast<int64_t>(out_row) * p.out_token + static_cast<int64_t>(out_head) * p.out_head;
#pragma unroll 1
      for (int c = 0; c < kVDim; c += 32) {
        uint32_t o[32];
        if (ran) {
          tmem_ld32(o_at + c, o);
          tmem_fence_ld(o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0;
        }
        if (twin) {
          uint32_t o1[32];
          tmem_ld32(o_col[1] + lanes + c, o1);
          tmem_fence_ld(o1);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            o[i] = __float_as_uint(__uint_as_float(o[i]) * own + __uint_as_float(o1[i]) * others);
        }
        if (repair && live) {
          // values that are not finite were taken out of the tiles that not
          // all rows see; a row that does see one gets it back: of its weight
          // it only counts whether it is zero
          const int ja = max(g.lim0, g.j0 * kTile), jb = min(lim, g.j1 * kTile);
          for (int j = ja; j < jb; ++j) {
            const uint16_t* v = static_cast<const uint16_t*>(p.vraw) +
                static_cast<int64_t>(g.k0 + j) * p.v_token + static_cast<int64_t>(g.head) * p.v_head +
                c;
            constexpr uint32_t kExp = kBf16 ? 0x7f80u : 0x7c00u, kFrac = kBf16 ? 0x7fu : 0x3ffu;
            uint32_t bad_ones = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) bad_ones |= static_cast<uint32_t>((v[i] & kExp) == kExp) << i;
            if (bad_ones == 0) continue;
            const bool none = no_weight<kDim, kBf16>(p, m, out_row, out_head, g.k0 + j, g.head);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (bad_ones >> i & 1u) {
                const uint32_t b = v[i];
                const float bad = none || (b & kFrac) ? __int_as_float(0x7fffffff)
                                  : (b & 0x8000u)     ? -INFINITY
                                                      : INFINITY;
                o[i] = __float_as_uint(__uint_as_float(o[i]) + bad);
              }
            }
          }
        }
        if (live && whole) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            w[i] = pack2<kBf16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
          if (p.wide) {
            store32(dst + c, w);
            store32(dst + c + 16, w + 8);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(dst + c + 8 * i) =
                  make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          }
        } else if (live) {
#pragma unroll
          for (int i = 0; i < 4; ++i) store32(part + c + 8 * i, o + 8 * i);
        }
        __syncwarp();
      }
      if (ran) {
        sl::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          sl::mbar_arrive(&sy.o_free[h]);
          if (twin) sl::mbar_arrive(&sy.o_free[1]);
        }
      }
    }
    // (the last turn that half 1 passed on)
    if (h == 0) take_turn();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  }
  if (warp == 8 || warp == 11) {
    // ------------------------------------------------- MMAs of one half
    const int h = warp == 8 ? 0 : 1;
    constexpr uint32_t idesc_s = idesc_f16(kBf16, kTile, false);
    constexpr uint32_t idesc_o = idesc_f16(kBf16, kVDim, true);
    const uint32_t q_lo = kKMajorLo + ((sl::smem_u32(buf) + h * C::kChunks * kSlotBytes) >> 4);
    const uint32_t ring_lo = sl::smem_u32(ring) >> 4;
    const uint32_t s_d = s_col[h], o_d = o_col[h];
    const bool leader = sl::elect_one();
    Tiles at;
    int n_o = 0;
    uint32_t clean_phase = 0;
    // S = Q K^T with the key tile at `at`, or (this half sees none of it) let
    // it go
    auto key_tile = [&](bool mine, bool last) {
      if (leader && out.ok) {
        if (mine) {
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c) {
            const uint32_t k_lo = kKMajorLo + ring_lo + at.place<C::kSlots>(c) * (kSlotBytes >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_ss(s_d, q_lo + c * (kSlotBytes >> 4) + 2 * k, k_lo + 2 * k, idesc_s, c + k > 0);
          }
          sl::umma_commit(&sy.s_full[h]);
          sl::umma_commit(&sy.empty[at.bar()]);
          // the next item's queries may come in while this one's last weights
          // are formed
          if (last) sl::umma_commit(&sy.q_empty[h]);
        } else {
          sl::mbar_arrive(&sy.empty[at.bar()]);
        }
      }
      __syncwarp();
      at.step<C::kSlots>(C::kChunks);
    };
    while (next_seg()) {
      uniform(g);
      if (g.j0 >= g.j1) continue;
      const bool twin = is_twin(g);
      const int j1 = twin ? g.j1 : min(g.j1, h ? g.nh[1] : g.nh[0]);
      const int j0 = twin ? g.j0 + h : g.j0;  // this half's first tile
      auto takes = [&](int j) { return twin ? ((j - j0) & 1) == 0 && j < j1 : j < j1; };
      const bool any = j0 < j1;
      if (any) out.wait(&sy.q_full[h], n_o & 1);
      out.wait(&sy.full[at.bar()], at.phase());
      sl::tc_fence_after();
      const int j_last = twin ? j1 - 1 - ((j1 - 1 - j0) & 1) : j1 - 1;
      key_tile(takes(g.j0), g.j0 == j_last);
      for (int j = g.j0; j < g.j1; ++j) {
        const bool mine = takes(j);
        // this tile's values and the next one's keys are here, as a rule, long
        // before the weights
        out.wait(&sy.full[at.bar()], at.phase());
        const int v_bar = at.bar();
        if ((j + 1) * kTile > g.lim0) {
          // cleaned by the guard first
          out.wait(&sy.clean[v_bar], (clean_phase >> v_bar) & 1);
          clean_phase ^= 1u << v_bar;
        }
        const int v_slot0 = at.place<C::kSlots>(0), v_slot1 = at.place<C::kSlots>(1);
        at.step<C::kSlots>(C::kVSlots);
        const bool next = j + 1 < g.j1;
        if (next) out.wait(&sy.full[at.bar()], at.phase());
        if (mine) {
          if (j == j0 && n_o > 0) out.wait(&sy.o_free[h], (n_o - 1) & 1);
          // O += P V in two halves of 64 keys, as the weights come in
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            bar_wait(kBarWeights + 2 * h + half, 160);
            sl::tc_fence_after();
            if (leader && out.ok) {
              const uint32_t v_lo = kRowMajorLo<C::kVRows> + ring_lo +
                  (C::kVSlots == 2 ? (half ? v_slot1 : v_slot0) * (kSlotBytes >> 4)
                                   : v_slot0 * (kSlotBytes >> 4) + half * 512);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_ts(o_d, s_d + 32 * half + 8 * k, v_lo + 128 * k, idesc_o,
                        j > j0 || half + k > 0);
            }
          }
          if (leader && out.ok) {
            sl::umma_commit(&sy.empty[v_bar]);
            sl::umma_commit(&sy.pv_done[h]);
          }
        } else if (leader && out.ok) {
          sl::mbar_arrive(&sy.empty[v_bar]);
        }
        __syncwarp();
        if (next) key_tile(takes(j + 1), j + 1 == j_last);
      }
      n_o += any;
    }
    // everything issued is in before TMEM and the barriers go
    if (leader) sl::umma_commit(&sy.drain[h]);
    __syncwarp();
    Outlook last;
    out.ok &= last.wait(&sy.drain[h], 0);
  } else if (warp == 9) {
    // ------------------------------------------------------------ loads
    Tiles at;
    // the oldest tile that still holds slots, whether it is one of values,
    // and the slots that are free
    uint32_t oldest = 0;
    bool oldest_v = false;
    int room = C::kSlots, n_q[2] = {0, 0};
    const uint32_t q_bytes = static_cast<uint32_t>(p.group * p.half_tokens) * 128;
    auto claim = [&](int slots) -> bool {
      while (room < slots) {
        if (!out.wait(&sy.empty[oldest % kBars], (oldest / kBars) & 1)) return false;
        room += oldest_v ? C::kVSlots : C::kChunks;
        oldest_v = !oldest_v;
        ++oldest;
      }
      room -= slots;
      if (lane == 0) sl::mbar_arrive_expect_tx(&sy.full[at.bar()], slots * kSlotBytes);
      return true;
    };
    while (next_seg()) {
      uniform(g);
      if (g.j0 >= g.j1) continue;
      auto load_q = [&](int h) -> bool {
        const bool twin = is_twin(g);
        if (g.j0 >= min(g.j1, h ? g.nh[1] : g.nh[0]) && !twin) return true;
        if (n_q[h] > 0 && !out.wait(&sy.q_empty[h], (n_q[h] - 1) & 1)) return false;
        ++n_q[h];
        if (lane == 0) {
          sl::mbar_arrive_expect_tx(&sy.q_full[h], q_bytes * C::kChunks);
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c)
            tma_load_3d(buf + (h * C::kChunks + c) * kSlotBytes, &p.q, &sy.q_full[h], 64 * c,
                        g.head * p.group, g.q0 + g.tok + (twin ? 0 : h * p.half_tokens));
        }
        return true;
      };
      auto load_k = [&](int j) -> bool {
        if (!claim(C::kChunks)) return false;
        if (lane == 0) {
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c) {
            // the last columns may be one row that all heads share
            const bool own = !(kDim == 192 && c == 2 && p.shared);
            tma_load_3d(ring + at.place<C::kSlots>(c) * kSlotBytes, own ? &p.k : &p.ks,
                        &sy.full[at.bar()], own ? 64 * c : 0, own ? g.head : 0,
                        g.k0 + j * kTile);
          }
        }
        at.step<C::kSlots>(C::kChunks);
        return true;
      };
      auto load_v = [&](int j) -> bool {
        if (!claim(C::kVSlots)) return false;
        if (lane == 0) {
#pragma unroll
          for (int i = 0; i < C::kVSlots; ++i)
#pragma unroll
            for (int c = 0; c < kVDim / 64; ++c)
              tma_load_3d(ring + at.place<C::kSlots>(i) * kSlotBytes + c * C::kVRows * 128, &p.v,
                          &sy.full[at.bar()], 64 * c, g.head, g.k0 + j * kTile + i * C::kVRows);
        }
        at.step<C::kSlots>(C::kVSlots);
        return true;
      };
      bool go = load_q(0) && load_k(g.j0) && load_q(1);
      for (int j = g.j0; j < g.j1 && go; ++j)
        go = load_v(j) && (j + 1 >= g.j1 || load_k(j + 1));
      if (!go) break;
    }
    if (!out.ok) {
      Outlook last;
      // what was asked for lands before the buffers go
      for (; oldest < at.n; ++oldest)
        last.wait(&sy.full[oldest % kBars], (oldest / kBars) & 1);
      for (int h = 0; h < 2; ++h)
        if (n_q[h] > 0) last.wait(&sy.q_full[h], (n_q[h] - 1) & 1);
    }
  } else if (warp == 10) {
    // ------------------------------------------------------- value guard
    // In a tile that reaches past what the item's first row sees, rows of
    // other sequences are zeroed (a weight of zero times what they hold could
    // be NaN), and so are values that are not finite; those that some row
    // does see are marked for the output to put back.
    Tiles at;
    int n_item = 0;
    Walk walk;
    walk.start(p, sy.cum);
    Seg ahead = {};
    auto publish = [&]() {
      const int i = n_seg % kSegs;
      if (n_seg >= kSegs && !out.wait(&sy.seg_empty[i], (n_seg / kSegs - 1) & 1)) return;
      if (!walk.next(p, sy.cum, per, ahead)) ahead.seq = -1;
      if (lane == 0) {
        sy.seg[i] = ahead;
        sl::mbar_arrive(&sy.seg_full[i]);
      }
      __syncwarp();
      ++n_seg;
    };
    // (one call in the loop: the lookup's code is fetched once)
    for (bool begun = false;; begun = true) {
      g = ahead;
      if (begun && (g.seq < 0 || !out.ok)) break;
      publish();
      if (!begun) {
        if (p.split && lane == 0) {
          const bool later = ahead.seq >= 0 && ahead.j0 > 0;
          Later w = {};
          w.unit0 = later ? walk.unit0 : -1;
          w.q0 = ahead.q0;
          w.q_len = ahead.q_len;
          w.k_len = ahead.k_len;
          w.tok = ahead.tok;
          w.head = ahead.head;
          p.later[blockIdx.x] = w;
        }
        continue;
      }
      uniform(g);
      if (g.j0 >= g.j1) continue;
      const int mark = n_item++;
      for (int j = g.j0; j < g.j1; ++j) {
        at.step<C::kSlots>(C::kChunks);
        // every value tile is waited for and let go, cleaned or not: a wait
        // names a use of its barrier by the parity alone
        if (!out.wait(&sy.full[at.bar()], at.phase())) break;
        if ((j + 1) * kTile > g.lim0) {
          bool found = false;
#pragma unroll 1
          for (int i = 0; i < C::kVSlots; ++i) {
            const int key0 = j * kTile + i * C::kVRows;
            const int lo = clampi(g.lim0 - key0, 0, C::kVRows);     // rows that all see
            const int hi = clampi(g.k_len - key0, 0, C::kVRows);    // rows of the sequence
            uint8_t* base = ring + at.place<C::kSlots>(i) * kSlotBytes;
            // (the slot's 64-column groups, one after the other)
#pragma unroll 1
            for (int c = 0; c < kVDim / 64; ++c)
              found |= clean_rows<kBf16>(base + c * C::kVRows * 128, lo, hi, C::kVRows, lane);
          }
          if (found) sy.mark[mark % kMarks] = mark;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) sl::mbar_arrive(&sy.clean[at.bar()]);
        }
        if (lane == 0) sl::mbar_arrive(&sy.empty[at.bar()]);
        at.step<C::kSlots>(C::kVSlots);
      }
    }
  }
  if (!out.ok && lane == 0) report(p, SL_ERR_TIMEOUT);
  sl::tc_fence_before();
  __syncthreads();
  sl::tc_fence_after();
  if (warp == 8) sl::tmem_dealloc(tmem, 512);
}

// Joins the partial results of an item that several CTAs share. Block c is the
// one to do it where CTA c holds an item's first stretch and CTA c + 1 a later
// one: in the order of the stretches, whatever order they were done in.
constexpr int kJoinThreads = 256;

template <int kVDim, bool kBf16>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(
    const __grid_constant__ Params p) {
  sl::pdl_wait();
  sl::pdl_trigger();
  constexpr unsigned kAll = 0xffffffffu;
  const int c = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Later g = p.later[c + 1];
  // CTAs c .. c + n - 1 have a stretch each
  int n = 1;
  for (int s0 = c;; s0 += 32) {
    const int unit = s0 + lane < p.grid ? p.later[s0 + lane].unit0 : -1;
    const unsigned other = __ballot_sync(kAll, unit != g.unit0 || unit < 0);
    if (s0 == c) {
      if (!(other & 1) || (other & 2)) return;  // not the first boundary inside an item
      n = (other >> 1) == 0 ? 32 : __ffs(other >> 1);
      if (n < 32) break;
    } else {
      n += other == 0 ? 32 : __ffs(other) - 1;
      if (other) break;
    }
  }
  const int rows = 2 * p.half_tokens * p.group;
  constexpr int kCols = kVDim / 32;  // of a lane
  constexpr int kAhead = 4;          // results of a row whose loads do not wait for its weights
  using Vec = typename std::conditional<kCols == 4, float4, float2>::type;
  const int step = gridDim.y * (kJoinThreads / 32);
  for (int r = blockIdx.y * (kJoinThreads / 32) + warp; r < rows; r += step) {
    const int token = r / p.group, tok = g.tok + token;
    if (tok >= g.q_len) break;
    const int lim = clampi(tok + 1 + g.k_len - g.q_len, 0, g.k_len);
    float m = -INFINITY, l = 0.f, o[kCols] = {};
    // the row of stretch s (of the first one's second slot, of the others' first)
    auto at = [&](int s) {
      return (2 * static_cast<int64_t>(c + s) + (s == 0)) * p.rows_cap + r;
    };
    auto load = [&](int s) {
      return reinterpret_cast<const Vec*>(p.part + at(s) * kVDim)[lane];
    };
    // a lane per stretch for the maxima and sums, then all lanes for the outputs
    for (int s0 = 0; s0 < n; s0 += 32) {
      const int here = min(32, n - s0);
      const float2 ml = lane < here ? p.part_ml[at(s0 + lane)] : make_float2(-INFINITY, 0.f);
      Vec v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (k < here) v[k] = load(s0 + k);
      float top = max2(m, ml.x);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) top = max2(top, __shfl_xor_sync(kAll, top, x));
      const float base = top == -INFINITY ? 0.f : top;
      const float mine = ex2((ml.x - base) * p.scale_log2), old = ex2((m - base) * p.scale_log2);
      float sum = lane < here ? ml.y * mine : 0.f;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(kAll, sum, x);
      l = l * old + sum;
      m = top;
#pragma unroll
      for (int i = 0; i < kCols; ++i) o[i] *= old;
      for (int k0 = 0; k0 < here; k0 += kAhead) {
        if (k0 > 0) {
#pragma unroll
          for (int k = 0; k < kAhead; ++k)
            if (k0 + k < here) v[k] = load(s0 + k0 + k);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const float w = __shfl_sync(kAll, mine, min(k0 + k, 31));
          if (k0 + k >= here) continue;
          const float* x = reinterpret_cast<const float*>(&v[k]);
#pragma unroll
          for (int i = 0; i < kCols; ++i) o[i] = fmaf(x[i], w, o[i]);
        }
      }
    }
    const float inv = lim == 0 ? 0.f : m == -INFINITY ? __int_as_float(0x7fffffff) : 1.f / l;
    uint16_t* dst = static_cast<uint16_t*>(p.out) +
        static_cast<int64_t>(g.q0 + tok) * p.out_token +
        static_cast<int64_t>(g.head * p.group + r - token * p.group) * p.out_head + lane * kCols;
#pragma unroll
    for (int i = 0; i < kCols; i += 2)
      *reinterpret_cast<uint32_t*>(dst + i) = pack2<kBf16>(o[i] * inv, o[i + 1] * inv);
  }
}

// --------------------------------------------------------------------- host
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

// [tokens, heads, columns] with strides in elements, in boxes of 64 columns
// (one 128-byte swizzled row each), box_heads heads and box_tokens tokens.
bool make_map(CUtensorMap* m, const void* base, bool bf16, int64_t columns, int64_t heads,
              int64_t tokens, int64_t head_stride, int64_t token_stride, int box_heads,
              int box_tokens) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(heads),
                        static_cast<cuuint64_t>(tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_stride) * 2,
                           static_cast<cuuint64_t>(token_stride) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  cuuint32_t step[3] = {1, 1, 1};
  return sl::encode_in_context([&] {
    return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
              const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

constexpr int64_t kHeaderBytes = 256;
constexpr int64_t kMostUnits = 1 << 22;

struct Shape {
  int64_t items, units;  // at most so many items, and key tiles of all items
  int64_t grid;
  bool split;
  int rows_cap;
};

Shape shape_of(int B, int64_t Tq, int64_t Tk, int heads, int kv_heads, int sms) {
  Shape r;
  const int group = heads / kv_heads;
  const int64_t tokens = 2 * (kTile / group);
  const int64_t items = (Tq + B * (tokens - 1)) / tokens;
  r.items = (items < Tq ? items : Tq) * kv_heads;
  r.units = r.items * (Tk / kTile + 1 + kItemUnits);
  const int64_t rows = Tq * group;
  r.rows_cap = static_cast<int>(rows < 2 * kTile ? rows : 2 * kTile);
  // Whole items, or equal shares of all key tiles and a join? In key tiles
  // (about 1.7 us each), for sequences of average length: whole items take as
  // long as the longest, as their even share, and, where all are about as long
  // (little of what they reach is their own diagonal), as their full turns;
  // shares take the even share and 6 for the join, 9 for one of full items.
  // Measured, shares against whole items in us: one token over 2048 keys of 4
  // heads 11.2 / 22.6, 8 over 512 12.0 / 10.4, 32 over 4096 52 / 47, 64 over
  // 2048 of 8 heads 92.5 / 96.3; 512 tokens behind 1024, 16 heads of 192, 26.9 /
  // 31.0, a prompt of 1024 28.0 / 24.1, of 8192 on 2 heads 48 / 109.
  const double longest = static_cast<double>(Tk) / B / kTile;
  const double seen = static_cast<double>(Tk) - 0.5 * static_cast<double>(Tq);
  const double average = (seen > 0 ? seen : 0) / B / kTile;
  const double even = r.items * (average + kItemUnits) / sms;
  double whole = longest + kItemUnits;
  if (even > whole) whole = even;
  if (4 * average >= 3 * longest) {
    const double turns = static_cast<double>((r.items + sms - 1) / sms) * (average + kItemUnits);
    if (turns > whole) whole = turns;
  }
  r.split = r.units < kMostUnits && even + (r.rows_cap < kTile ? 6 : 9) < whole;
  r.grid = r.split ? (r.units < sms ? r.units : sms) : (r.items < sms ? r.items : sms);
  return r;
}

template <int kDim, int kVDim, bool kBf16>
int launch_all(const Params& p, cudaStream_t st) {
  auto kern = attention_kernel<kDim, kVDim, kBf16>;
  static std::atomic<uint64_t> smem_set{0};
  SL_CUDA_TRY(sl::ensure_smem_limit(kern, kSmemBytes, smem_set));
  SL_CUDA_TRY(sl::launch(kern, dim3(p.grid), dim3(kThreads), kSmemBytes, st, p));
  if (p.split && p.grid > 1)
    SL_CUDA_TRY(sl::launch(attention_join_kernel<kVDim, kBf16>,
                           dim3(p.grid - 1, (p.rows_cap + 31) / 32), dim3(kJoinThreads), 0, st,
                           p));
  return SL_OK;
}

}  // namespace

extern "C" size_t sl_prompt_attention_workspace_bytes(int B, int64_t Tq, int64_t Tk, int heads,
                                                      int kv_heads, int v_dim) {
  if (B <= 0 || Tq < 0 || Tk < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads ||
      heads / kv_heads > kTile || v_dim <= 0)
    return 0;
  const int sms = sl_device_sm_count();
  // (without a device: the size for this part's 148)
  const Shape r = shape_of(B, Tq, Tk, heads, kv_heads, sms > 0 ? sms : 148);
  if (!r.split) return kHeaderBytes;
  return static_cast<size_t>(kHeaderBytes + r.grid * static_cast<int64_t>(sizeof(Later)) +
                             2 * r.grid * r.rows_cap * (4 * static_cast<int64_t>(v_dim) + 8));
}

extern "C" int sl_prompt_attention(const sl_attention_args* args, void* workspace,
                                   size_t workspace_bytes, sl_stream_t stream) {
  return sl_prompt_attention_ex(args, workspace, workspace_bytes, nullptr, stream);
}

extern "C" int sl_prompt_attention_ex(const sl_attention_args* args, void* workspace,
                                      size_t workspace_bytes, int32_t* failed,
                                      sl_stream_t stream) {
  if (!args) return SL_ERR_INVALID;
  const sl_attention_args& a = *args;
  if (a.B <= 0 || a.Tq < 0 || a.Tk < 0 || a.heads <= 0 || a.kv_heads <= 0 ||
      a.heads % a.kv_heads || !(a.scale > 0.f) || !(a.scale < INFINITY) || a.shared_dim < 0)
    return SL_ERR_INVALID;
  const bool dims = (a.dim == 64 && a.v_dim == 64) || (a.dim == 128 && a.v_dim == 128) ||
                    (a.dim == 192 && a.v_dim == 128);
  if (!dims || (a.shared_dim != 0 && !(a.shared_dim == 64 && a.dim == 192)) ||
      (a.dtype != SL_DTYPE_BF16 && a.dtype != SL_DTYPE_FP16) || a.heads / a.kv_heads > kTile ||
      a.Tq > 0x7fffffff || a.Tk > 0x7fffffff)
    return SL_ERR_UNSUPPORTED;
  if (a.Tq == 0) return SL_OK;
  const bool keys = a.Tk > 0;
  if (!a.q || !a.out || !a.cu_q || !a.cu_k || !workspace || (keys && (!a.k || !a.v)) ||
      (keys && a.shared_dim && !a.k_shared))
    return SL_ERR_INVALID;
  if (workspace_bytes < sl_prompt_attention_workspace_bytes(a.B, a.Tq, a.Tk, a.heads, a.kv_heads,
                                                            a.v_dim))
    return SL_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
       reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.k_shared) |
       reinterpret_cast<uintptr_t>(a.out)) & 15 || (reinterpret_cast<uintptr_t>(workspace) & 31))
    return SL_ERR_INVALID;
  if ((a.q_token | a.q_head | a.k_token | a.k_head | a.v_token | a.v_head | a.k_shared_token |
       a.out_token | a.out_head) & 7)
    return SL_ERR_INVALID;
  const int sms = sl_device_sm_count();
  if (sms <= 0) return SL_ERR_CUDA;
  const Shape r = shape_of(a.B, a.Tq, a.Tk, a.heads, a.kv_heads, sms);
  if (r.items >= kMostUnits) return SL_ERR_UNSUPPORTED;
  const bool bf16 = a.dtype == SL_DTYPE_BF16;
  Params p = {};
  p.group = a.heads / a.kv_heads;
  p.half_tokens = kTile / p.group;
  bool ok = make_map(&p.q, a.q, bf16, a.dim, a.heads, a.Tq, a.q_head, a.q_token, p.group,
                     p.half_tokens);
  if (keys) {
    ok = ok && make_map(&p.k, a.k, bf16, a.dim - a.shared_dim, a.kv_heads, a.Tk, a.k_head,
                        a.k_token, 1, kTile);
    ok = ok && make_map(&p.v, a.v, bf16, a.v_dim, a.kv_heads, a.Tk, a.v_head, a.v_token, 1,
                        a.v_dim == 128 ? kTile / 2 : kTile);
    if (a.shared_dim)
      ok = ok && make_map(&p.ks, a.k_shared, bf16, a.shared_dim, 1, a.Tk, a.shared_dim,
                          a.k_shared_token, 1, kTile);
  }
  if (!ok) return SL_ERR_INVALID;
  p.out = a.out;
  p.out_token = a.out_token;
  p.out_head = a.out_head;
  p.cu_q = a.cu_q;
  p.cu_k = a.cu_k;
  p.vraw = a.v;
  p.v_token = a.v_token;
  p.v_head = a.v_head;
  p.qraw = a.q;
  p.q_token = a.q_token;
  p.q_head = a.q_head;
  p.kraw = a.k;
  p.k_token = a.k_token;
  p.k_head = a.k_head;
  p.ksraw = a.shared_dim ? a.k_shared : nullptr;
  p.ks_token = a.k_shared_token;
  p.B = a.B;
  p.Tq = static_cast<int>(a.Tq);
  p.Tk = static_cast<int>(a.Tk);
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.shared = a.shared_dim != 0;
  p.wide = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0 && ((a.out_token | a.out_head) & 15) == 0;
  p.grid = static_cast<int>(r.grid);
  p.split = r.split;
  p.rows_cap = r.rows_cap;
  auto divisor = [](int d) {
    Divisor v = {0, 0, d};
    while ((1 << v.shift) < d) ++v.shift;
    v.mul = static_cast<uint32_t>(((1ull << (31 + v.shift)) + d - 1) / d);
    return v;
  };
  p.by_tokens = divisor(2 * p.half_tokens);
  p.by_heads = divisor(p.kv_heads);
  p.by_grid = divisor(p.grid);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.lag = (bf16 ? kLagBf16 : kLagF16) / p.scale_log2;
  p.status = static_cast<int32_t*>(workspace);
  p.failed = failed;
  p.later = reinterpret_cast<Later*>(static_cast<uint8_t*>(workspace) + kHeaderBytes);
  p.part = reinterpret_cast<float*>(p.later + r.grid);
  p.part_ml = reinterpret_cast<float2*>(p.part + 2 * r.grid * r.rows_cap * a.v_dim);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a.dim == 64) return bf16 ? launch_all<64, 64, true>(p, st) : launch_all<64, 64, false>(p, st);
  if (a.dim == 128)
    return bf16 ? launch_all<128, 128, true>(p, st) : launch_all<128, 128, false>(p, st);
  return bf16 ? launch_all<192, 128, true>(p, st) : launch_all<192, 128, false>(p, st);
}
