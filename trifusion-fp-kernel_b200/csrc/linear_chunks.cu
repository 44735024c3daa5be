// Linear attention with a decay for each head: the chunked form for prompts.
//
// Chunk of C = 64 tokens, state S (N x P) before it, c_i = g_1 + .. + g_i within it:
//
//   o_i   = scale * ( e^{c_i} q_i S  +  sum_{j <= i} e^{c_i - c_j} (q_i . k_j) v_j )
//   S'    = e^{c_C} S + sum_j k_j (e^{c_C - c_j} v_j)^T
//
// Everything with a token pair or a state element in it is a 64-token matrix
// product on the tensor cores (tcgen05, BF16 operands, FP32 accumulators in TMEM),
// with the value dimension on the 128 accumulator lanes:
//
//   D [i, j]     = q k^T                       M 64   N 64   K N
//   dS^T [p, n]  = (w v)^T k, w_j = e^{c_C-c_j}  M 128  N N    K 64, three times
//   OI^T [p, i]  = S^T q^T                     M 128  N 64   K N
//   OP^T [p, i]  = v^T P^T, P = D e^{c_i-c_j}  M 128  N 64   K 64, once a head
//
// The 128 lanes are two blocks of 64 value columns: the two halves of one wide head
// (P > 64), or two heads (P <= 64) that share a k head, so that their D is formed
// once and their state updates are one product.
//
// Precision. q, k and v enter the products as they are (BF16). w v is split into
// three BF16 parts whose sum holds its 24 bits, so the state and its FP32 update are
// as exact as an FP32 product; S lives in FP32 registers. Two roundings to BF16 are
// made on the way to the output: P (after the decay) and S as the operand of q S.
// Each is half a step of a term, like the output's own rounding. The sums of decays
// of the state's weights run from the chunk's end (exact where they matter), the
// ones of e^{c_i} from its start.
//
// Long rows on few heads: the time axis is cut into segments. One launch forms every
// segment's own state from zero, one joins them (S_in of each segment), and the main
// launch runs all segments side by side.
//
// One CTA of 32 warps an SM, a warp for each step and mbarriers between the steps, so that
// several chunks are in work at once: loads (TMA), decay sums, weighted values, scores to P,
// outputs, the state, and one warp each for the products that need the state before and those
// that do not. What decides: 64 registers a thread (shared out again by setmaxnreg) and code that
// stays in the instruction cache - loops are kept rolled where unrolling them cost a fetch a pass.
// Measured on a B200 (device time; copy rate 6552 GB/s):
//   2 x 26 tokens, 4 heads, N 128, P 64        9.0 us   launch, set-up and two memory latencies
//   16 x 200 ragged, 12 heads, N 128, P 64    14.3 us   four chunks in a row of about 2400 cycles
//   2 x 3600 ragged, 12 heads, N 128, P 64    34.9 us   5 chunks a segment, twice, and a join
//   1 x 32768, 16 + 16 heads, 128 x 128      168 us     102 us at 5.1 TB/s, 58 us for the
//                                                       segments' states (4.1 TB/s), join 8 us
//   8 x 4097 ragged, 32 + 8 heads, 64 x 64    91 us     issue: 73 % of the slots of 128 SMs
//   24 x 3600, 12 heads, N 128, P 64         100 us     144 CTAs, 57 chunks each
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>

#include "../../include/trifusion_b200.h"
#include "linear_attention.cuh"
#include "sm100.cuh"
#include "tf_host.cuh"

namespace tf {
namespace {
using namespace sm100;

constexpr int kC = 64;                // tokens of a chunk
constexpr int kBox = 8192;            // bytes of a 64 x 64 BF16 tile
constexpr int kSums = 4;              // chunks whose decay sums are kept
// A decay below it is zero in FP32 against any state. (64 of them in a chunk add up to 2^14,
// where the sums' steps are 2^-10: weights within 2^-10 or so, less than P's rounding.)
constexpr float kMinLog2 = -256.f;
// In place of a state's factor that is zero in FP32, so that an infinite state stays infinite.
constexpr float kTiny = 0x1p-149f;

// Warps, by what they do; groups of four have the four quarters of the TMEM lanes, pairs of
// groups the two halves of a chunk's tokens.
constexpr int kPrepWarp = 4, kScoreWarp = 12, kOutWarp = 20;  // (state: 0)
// A quarter's warps share a scheduler, and the later a chunk's rows the more scores they have:
// the last quarter's gets the lightest of the single warps (100 -> 92 us for 8 x 4097 tokens,
// with the sums of both heads in one pass).
constexpr int kSumWarp = 28, kStateMmaWarp = 29, kOutMmaWarp = 30, kLoadWarp = 31;
constexpr int kThreads = 32 * 32;
// Registers of a thread: 32 warps have 64 at launch, 2048 together, and share them out again.
// The state's four warps hold 64 or 128 values a thread. (What the compiler spills hangs on these
// numbers in no simple way: with 168 for the state of N > 64 it is 200 to 300 bytes a thread of other
// warps.) A wide segment's own state has no scores, and spills nothing with their registers.
template <int NK, bool WIDE, bool FULL>
struct Regs {
  static constexpr bool own = NK == 2 && WIDE && !FULL;
  static constexpr int state = NK == 1 ? 120 : own ? 200 : 152, prep = NK == 1 ? 56 : 48,
                       score = NK == 1 ? 56 : own ? 24 : 48, out = 56, single = 56;
  static_assert(4 * state + 8 * (prep + score + out) + 4 * single == 2048, "what was launched");
};

constexpr int kLinearGaveUp = 3;      // (1 and 2 are the recurrence kernels')
__device__ int g_linear_error = 0;    // kLinearGaveUp: a bounded wait gave up

struct ChunkParams {
  CUtensorMap tm_q, tm_k, tm_v, tm_o;
  LinearParams l;
  int pairs;       // CTAs of a k head: pairs of its heads (P <= 64), or its heads
  int segs;        // segments of the time axis
  int seg_chunks;  // chunks of a segment
  float* seg_state;   // [B*H][segs][N][P]: the state before each segment
  float* seg_decay;   // [B*H][segs]: log2 decay over the segment
  int* err_host;
  uint32_t tries;     // limit of the kernel's waits
};

// What a CTA works on. Its warps read it from shared memory where they start: few of them
// have registers for all of it.
struct alignas(16) Unit {
  int b, hk, seg;      // row, k head, segment
  int head0, nheads;   // v heads: one (wide, or without a partner) or two
  int len;             // the row's length
  int first, last;     // its chunks with live tokens
  int64_t slot;        // of the row's state
  __device__ __forceinline__ int live(int it) const { return min(len - (first + it) * kC, kC); }  // tokens of a chunk
  __device__ __forceinline__ bool ends_row() const { return last == (len + kC - 1) / kC; }
};
template <int STAGES>
struct alignas(16) Misc {
  Unit unit;
  uint64_t full[STAGES], empty[STAGES];      // tiles loaded / every product of them done
  uint64_t sums[kSums], sums_free[kSums];    // decay sums written / read
  uint64_t d_full[2];                        // scores there
  uint64_t p_ready[2], o_full[2];            // P written, both output products there
  uint64_t oi_free, op_free[2];              // the products read
  uint64_t wv_ready[2][2], wv_free[2][2];    // [buffer][half] weighted values written / read
  uint64_t ds_full[2], ds_free[2];           // state product there / read
  uint64_t s_ready, s_free;                  // state operand written / read
  uint64_t init_full, init_read;             // the state before the first chunk there / read
  uint64_t drained[2];                       // a product warp's last product and arrivals are done
  uint32_t tmem;
  alignas(16) float row[kSums][2][kC];  // [chunk][head] two factors of scale e^{c_i - c_j}, or c_i and
  float col[kSums][2][kC];              // -c_j (log2) where a factor would leave FP32's range
  float ecs[kSums][2][kC];              // scale e^{c_i}
  float w[kSums][2][kC];                // e^{c_C - c_j}, 0 past the length
  float total[kSums][2];                // e^{c_C}, below zero where a decay is -inf
  int factors[kSums][2];                // row and col hold factors
  int reset[kSums][2];                  // the first token with a decay of -inf, where there is one
};
// Shared memory, in bytes from a 1024-byte boundary: as many stages (chunks) as fit, up to
// six. The value tiles of a pair of heads lie around one zero tile, .. a1 a0 zero b0 b1 ..: a
// head's tile and the zero tile are the two 64-column blocks of the operand of its OP product.
template <int NK, bool WIDE, bool FULL>
struct Layout {
  static constexpr int tiles = (FULL ? 2 : 1) * NK + 2;     // of a stage
  static constexpr int fixed = FULL ? (WIDE ? 2 : 5) * kBox + 8 * 2048 : 0;
  static constexpr int fit = (232448 - 1024 - static_cast<int>(sizeof(Misc<6>)) - fixed) / (tiles * kBox);
  static constexpr int stages = fit > 6 ? 6 : fit;
  static constexpr bool zero_tile = FULL && !WIDE;
  static constexpr int k = 0;                               // [stage][NK]
  static constexpr int q = k + stages * NK * kBox;          // [stage][NK]
  static constexpr int v = q + (FULL ? stages * NK * kBox : 0);
  static constexpr int zero = v + stages * kBox;
  static constexpr int p = v + (2 * stages + (zero_tile ? 1 : 0)) * kBox;  // [chunk & 1][head]
  static constexpr int o = p + (FULL ? (WIDE ? 2 : 4) * kBox : 0);         // [warp] 32 tokens x 32 columns
  static constexpr int misc = o + (FULL ? 8 * 2048 : 0);
  // Two areas of up to 32 KB for states: before the first chunk in the stages after its own,
  // at the end anywhere.
  static constexpr int init0 = k + NK * kBox, init1 = q + NK * kBox, last0 = 0, last1 = 32768;
  static_assert(!FULL || (stages - 1) * NK * kBox >= 16384 * NK, "room for the states");
  static constexpr int bytes = misc + static_cast<int>(sizeof(Misc<stages>)) + 1024;
  static_assert(stages >= 3 && bytes <= 232448, "shared memory of a CTA");
  static __device__ __forceinline__ uint32_t va(int stage) {
    return zero_tile ? zero - (stage + 1) * kBox : v + 2 * stage * kBox;
  }
  static __device__ __forceinline__ uint32_t vb(int stage) {
    return zero_tile ? zero + (stage + 1) * kBox : v + (2 * stage + 1) * kBox;
  }
  static __device__ __forceinline__ uint32_t ptile(int it, int head) {
    return p + (WIDE ? it & 1 : 2 * (it & 1) + head) * kBox;
  }
};
// The stage of a chunk and the parity of its turn there.
template <int STAGES>
struct Ring {
  int st = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++st == STAGES) st = 0, ph ^= 1;
  }
};

// TMEM columns. The weighted values (three parts of 64 tokens) and the state (BF16) are
// operands there: as shared-memory tiles they would cost 160 KB of its traffic a chunk.
// D and then OP of a chunk share 64 columns, and neighbouring chunks have two sets of them,
// so that one's D is formed while the other's OP is read. What the 512 columns leave room for
// is held twice as well: the weighted values where N <= 64; for a segment's own state, its
// weighted values and products.
template <int NK, bool FULL>
struct Tmem {
  static constexpr int wv_bufs = FULL && NK == 2 ? 1 : 2, ds_bufs = FULL ? 1 : 2;
  static constexpr uint32_t x = 0, ds = FULL ? 128 : 0, oi = ds + 64 * NK * ds_bufs, wv = oi + (FULL ? 64 : 0),
                            s = wv + 96 * wv_bufs, end = s + (FULL ? 32 * NK : 0);
  static_assert(end <= 512, "TMEM has 512 columns");
};

constexpr uint32_t idesc_bf16(int m, int n, bool a_mn, bool b_mn) {
  return idesc_f16_f32(m, n, a_mn, b_mn) | (1u << 7) | (1u << 10);
}

__device__ __forceinline__ bool bar_or(int id, int n, bool x) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, %3, p;\n"
      " selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(x)), "r"(id), "r"(n)
      : "memory");
  return r != 0;
}
// Waits for the phase with `parity` to complete; false after `tries` tries and one. A try suspends the
// thread for up to 4 us (kTryNs, measured). Counted, not timed: the waits are a part of the code that
// every warp fetches; with a clock in each of them 24 x 3600 tokens of 12 heads (N 128, P 64) took 122 us,
// not 97.
constexpr uint32_t kTryNs = 4000, kTries = 2000000000u / kTryNs;
__device__ __forceinline__ bool wait_tries(uint64_t* bar, uint32_t parity, uint32_t tries = kTries) {
  for (uint32_t i = 0; !mbar_try_wait(bar, parity); ++i)
    if (i >= tries) return false;
  return true;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("{\n .reg .b64 st;\n mbarrier.arrive.shared::cta.b64 st, [%0];\n}\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void sts4(uint32_t a, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
// Four 8 x 8 fragments stored transposed: lane l gives the address of row l % 8 of matrix l / 8.
__device__ __forceinline__ void stsm_x4_t(uint32_t a, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(r0), "r"(r1),
               "r"(r2), "r"(r3)
               : "memory");
}
__device__ __forceinline__ void tma_store_4d(const void* tmap, uint32_t src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(reinterpret_cast<uint64_t>(dst)),
               "r"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
// 16 lanes x 8 columns: thread t gives lanes t/4 and t/4 + 8, column 4 x + t % 4, as r[2 x]
// and r[2 x + 1].
__device__ __forceinline__ void tmem_st_16x128_x2(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}
// A lane's 16 consecutive columns.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st1(uint32_t taddr, uint32_t r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(r) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 16 TMEM lanes x 16 columns as m16n8 fragments: thread t gets lanes t/4 and t/4 + 8,
// columns 8 x + 2 (t % 4) + {0, 1}, as r[4 x + 0..1] and r[4 x + 2..3].
__device__ __forceinline__ void tmem_ld_frag2(uint32_t taddr, float (&r)[8]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
               : "r"(taddr)
               : "memory");
}
// The two halves of a shared-memory descriptor (sm100.cuh's desc_sw128 with 8-row groups of
// 1024 bytes): the upper one is the same for all, the lower one has address and lbo.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | (lbo >> 4 << 16); }
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) {
  return static_cast<uint64_t>((1024u >> 4) | (1u << 14) | (2u << 29)) << 32 | lo;
}
// D[tmem] (+)= A[tmem] * B[smem].
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One lane of a converged warp; the code around it stays uniform.
__device__ __forceinline__ bool elect_one() {
  uint32_t x;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(x));
  return x != 0;
}
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// The upper halves of x (their first 8 significant bits) as a BF16 pair, taken off x. Twice,
// then what is left has 8 bits or fewer: three pairs hold 24 bits exactly.
__device__ __forceinline__ uint32_t take_bf16(float2& x) {
  const uint32_t a = __float_as_uint(x.x), b = __float_as_uint(x.y);
  x = fma2(make_float2(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u)), make_float2(-1.f, -1.f), x);
  return __byte_perm(a, b, 0x7632);
}

template <bool WIDE>
__device__ __forceinline__ Unit unit_of(const ChunkParams& p, int x) {
  Unit u;
  const LinearParams& l = p.l;
  u.seg = x % p.segs;
  x /= p.segs;
  const int pr = x % p.pairs;
  x /= p.pairs;
  u.hk = x % l.Hq;
  u.b = x / l.Hq;
  const int share = l.H / l.Hq;
  u.head0 = u.hk * share + (WIDE ? pr : 2 * pr);
  u.nheads = WIDE || 2 * pr + 1 >= share ? 1 : 2;
  u.len = l.T;
  if (l.lengths) u.len = static_cast<int>(min(max(l.lengths[u.b], static_cast<int64_t>(0)), static_cast<int64_t>(l.T)));
  u.first = u.seg * p.seg_chunks;
  u.last = min((u.len + kC - 1) / kC, u.first + p.seg_chunks);
  u.slot = l.slots ? l.slots[u.b] : u.b;
  return u;
}

// Output rows of a CTA from t0 on, as far as its segment goes: zeros, or `word` before the length.
__device__ __forceinline__ void fill_rows(const ChunkParams& p, const Unit& u, int t0, int thread, int threads,
                                       uint32_t word) {
  const LinearParams& l = p.l;
  const int t1 = static_cast<int>(min(static_cast<int64_t>(l.T), static_cast<int64_t>(u.first + p.seg_chunks) * kC));
  if (t0 >= t1) return;
  const int vecs = u.nheads * l.P / 8, rows = threads / vecs;  // 16-byte vectors of a token; tokens at a time
  const int c = thread % vecs * 8;
  bf16* o = static_cast<bf16*>(l.out) + u.b * l.so[0] + (u.head0 + c / l.P) * l.so[2] + c % l.P;
  if (thread < rows * vecs)
    for (int64_t t = t0 + thread / vecs; t < t1; t += rows) {
      const uint32_t x = t < u.len ? word : 0u;
      *reinterpret_cast<uint4*>(o + t * l.so[1]) = make_uint4(x, x, x, x);
    }
}

// FULL: the outputs and the final state; otherwise a segment's own state from zero.
template <int NK, bool WIDE, bool FULL>
__global__ void __launch_bounds__(kThreads, 1) linear_chunk_kernel(const __grid_constant__ ChunkParams p) {
  using L = Layout<NK, WIDE, FULL>;
  constexpr int kStages = L::stages;
  using C = Tmem<NK, FULL>;
  using R = Regs<NK, WIDE, FULL>;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t sb = (smem_u32(smem_raw) + 1023u) & ~1023u;
  Misc<kStages>& m = *reinterpret_cast<Misc<kStages>*>(smem_raw + (sb - smem_u32(smem_raw)) + L::misc);
  const LinearParams& l = p.l;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // Waits of the kernel's steps for one another. One that gives up ends its warp's work: the warps
  // behind it give up too, the copies and products already issued are waited for (with a limit that
  // is fixed), TMEM is freed, and the launch leaves an error and invalid outputs and states.
  auto wait_for = [&](uint64_t* bar, uint32_t parity) { return wait_tries(bar, parity, p.tries); };
  // The states of this CTA's heads lie in pieces of neighbouring values: 64 rows at a time of
  // one wide head, or the heads of a pair.
  auto pieces = [&](const Unit& u) { return WIDE ? NK : u.nheads; };
  auto piece_bytes = [&](int x) { return static_cast<uint32_t>((WIDE ? min(l.N - 64 * x, 64) : l.N) * l.P * 4); };
  auto seg_piece = [&](const Unit& u, int seg, int x) {
    const int64_t row = static_cast<int64_t>(u.b) * l.H + u.head0 + (WIDE ? 0 : x);
    return p.seg_state + (row * p.segs + seg) * (static_cast<int64_t>(l.N) * l.P) + (WIDE ? x * 64 * l.P : 0);
  };
  auto pool_piece = [&](const Unit& u, int x) {
    return l.state + u.slot * l.ss[0] + (u.head0 + (WIDE ? 0 : x)) * l.ss[1] + (WIDE ? x * 64 * l.P : 0);
  };
  const bool has_init = FULL && (p.segs > 1 || (l.state && !l.fresh));
  // Decays of this lane's tokens of a chunk: a head has all lanes of a warp, or each of two
  // heads half of them; a lane has kT neighbouring tokens.
  constexpr int kT = WIDE ? 2 : 4, kLanes = kC / kT;
  auto load_decays = [&](const Unit& u, int it, float* to) {
    const int x = lane / kLanes, t = (u.first + it) * kC + lane % kLanes * kT;
    const float* g = l.decay + u.b * l.sg[0] + (u.head0 + x) * l.sg[1];
#pragma unroll
    for (int j = 0; j < kT; ++j)
      to[j] = x < u.nheads && t + j < u.len ? g[static_cast<int64_t>(t + j) * l.sg[2]] : 0.f;
  };
  // One chunk's tiles into a stage.
  auto load_chunk = [&](const Unit& u, int it, int st) {
    const bool two = WIDE || u.nheads == 2;  // the second block of value columns is there
    const int t = (u.first + it) * kC;
    mbar_arrive_expect_tx(&m.full[st], ((FULL ? 2 : 1) * NK + (two ? 2 : 1)) * kBox);
    for (int x = 0; x < NK; ++x) {
      tma_load_4d(sb + L::k + (st * NK + x) * kBox, &p.tm_k, &m.full[st], 64 * x, u.hk, t, u.b);
      if (FULL) tma_load_4d(sb + L::q + (st * NK + x) * kBox, &p.tm_q, &m.full[st], 64 * x, u.hk, t, u.b);
    }
    tma_load_4d(sb + L::va(st), &p.tm_v, &m.full[st], 0, u.head0, t, u.b);
    if (two)
      tma_load_4d(sb + L::vb(st), &p.tm_v, &m.full[st], WIDE ? 64 : 0, WIDE ? u.head0 : u.head0 + 1, t, u.b);
  };
  // ---- set-up ------------------------------------------------------------------
  const Unit first_unit = unit_of<WIDE>(p, blockIdx.x);
  float decays[4] = {};  // the sum warp's first ones, on their way while the rest is set up
  {
    const Unit& u = first_unit;
    bool dead = false;  // no state of its own: padding, a wrong slot, or one that an earlier row has
    if (FULL) dead = l.state && (u.slot < 0 || u.slot >= l.nslots);
    const bool idle = dead || u.first >= u.last || (!FULL && u.ends_row());
    if (warp == kLoadWarp) {
      if (lane == 0) {
        m.unit = u;
        for (int i = 0; i < kStages; ++i) {
          mbar_init(&m.full[i], 1);
          mbar_init(&m.empty[i], FULL ? 2 : 1);
        }
        for (int i = 0; i < kSums; ++i) {
          mbar_init(&m.sums[i], 1);
          mbar_init(&m.sums_free[i], FULL ? 12 : 4);
        }
        for (int i = 0; i < 2; ++i) {
          mbar_init(&m.p_ready[i], 8);
          mbar_init(&m.o_full[i], 1);
          mbar_init(&m.op_free[i], 8);
          mbar_init(&m.d_full[i], 1);
          for (int j = 0; j < 2; ++j) {
            mbar_init(&m.wv_ready[i][j], 4);
            mbar_init(&m.wv_free[i][j], 1);
          }
          mbar_init(&m.ds_full[i], 1);
          mbar_init(&m.ds_free[i], 4);
        }
        mbar_init(&m.drained[0], 1);
        mbar_init(&m.drained[1], 1);
        mbar_init(&m.oi_free, 8);
        mbar_init(&m.s_ready, 4);
        mbar_init(&m.s_free, 1);
        mbar_init(&m.init_full, 1);
        mbar_init(&m.init_read, 4);
        fence_mbar_init();
      }
      __syncwarp();
    } else if (warp == kStateMmaWarp) {
      tmem_alloc(&m.tmem, 512);
      tmem_relinquish();
    }
    if (warp == kSumWarp && !idle) load_decays(u, 0, decays);
    if (FULL && l.slots)
      for (int i = tid; i < u.b; i += kThreads) dead |= l.slots[i] == u.slot;
    tc_fence_before();
    dead = __syncthreads_or(dead);
    tc_fence_after();
    if (dead || idle) {
      // Nothing to work on, or (a segment's own state) nobody who would read it.
      if (FULL) fill_rows(p, u, u.first * kC, tid, kThreads, dead && u.slot >= 0 ? 0x7fc07fc0u : 0u);
      if (FULL && !dead && u.len == 0 && u.seg == 0 && l.fresh && l.state)
        for (int i = tid; i < u.nheads * l.N * l.P; i += kThreads)
          l.state[u.slot * l.ss[0] + (u.head0 + i / (l.N * l.P)) * l.ss[1] + i % (l.N * l.P)] = 0.f;
      if (warp == kStateMmaWarp) tmem_dealloc(m.tmem, 512);
      return;
    }
  }
  const uint32_t tm = m.tmem;
  const int q4 = warp & 3;                  // quarter of the TMEM lanes
  const uint32_t tl = (32u * q4) << 16;
  bool bad = false;  // a bounded wait gave up

  if (warp >= kSumWarp) {
    fewer_registers<R::single>();
    const Unit u = m.unit;
    const int n_chunks = u.last - u.first;
    // A product warp ends when its products and their arrivals at barriers are done: none may still
    // be on its way into shared memory or TMEM when the CTA gives them up.
    auto drain = [&](int x) {
      if (elect_one()) umma_commit(&m.drained[x]);
      __syncwarp();
      return __all_sync(0xffffffffu, wait_tries(&m.drained[x], 0)) != 0;
    };
    if (warp == kLoadWarp && lane == 0) {
      // ---- loads ----------------------------------------------------------------
      int issued = 0;
      Ring<kStages> ring;
      for (int it = 0; it < n_chunks; ++it, ring.next()) {
        // The stages after the first are free once the state has been taken out of them.
        // (A limit of less than one try: the first wait gives up, and all that wait for its tiles do.)
        const bool first = it == 1 && has_init, later = it >= kStages;
        if ((first || later) && p.tries == 0 || first && !wait_for(&m.init_read, 0) ||
            later && !wait_for(&m.empty[ring.st], ring.ph ^ 1)) {
          bad = true;
          break;
        }
        load_chunk(u, it, ring.st);
        ++issued;
        if (it == 0 && has_init) {
          uint32_t bytes = 0;
          for (int x = 0; x < pieces(u); ++x) bytes += piece_bytes(x);
          mbar_arrive_expect_tx(&m.init_full, bytes);
          for (int x = 0; x < pieces(u); ++x)
            bulk_load(sb + (x ? L::init1 : L::init0), p.segs > 1 ? seg_piece(u, u.seg, x) : pool_piece(u, x),
                      piece_bytes(x), &m.init_full);
        }
      }
      // No copy of this CTA may be in flight when it ends (also after a wait that gave up).
      for (int i = max(0, issued - kStages); i < issued; ++i) bad |= !wait_tries(&m.full[i % kStages], (i / kStages) & 1);
      if (has_init) bad |= !wait_tries(&m.init_full, 0);
    } else if (warp == kStateMmaWarp) {
      // ---- products that need nothing of the state before --------------------------
      // The whole warp runs this, one lane issues: addresses stay in uniform registers.
      // (Two warps for the products: with one, its waits and issue were the longest path.)
      // The lanes wait for themselves, and stopping is one decision of the warp, once a chunk: lanes that
      // left alone would keep the others at elect for good. Until then the products run on whatever
      // is there; the launch's results are invalid then anyway.
      Ring<kStages> ring;
      bool ok = true;
      auto scores = [&](int it) {  // D
        const int st = ring.st;
        ok &= wait_for(&m.full[st], ring.ph);
        if (it >= 2) ok &= wait_for(&m.op_free[it & 1], ((it >> 1) - 1) & 1);
        tc_fence_after();
        const uint32_t qd = desc_lo(sb + L::q + st * NK * kBox, 0), kd = desc_lo(sb + L::k + st * NK * kBox, 0);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4 * NK; ++kk) {
            const uint32_t off = ((kk >> 2) * kBox + (kk & 3) * 32u) >> 4;
            umma_f16(tm + C::x + 64 * (it & 1), desc_of(qd + off), desc_of(kd + off), idesc_bf16(64, 64, false, false), kk > 0);
          }
          umma_commit(&m.d_full[it & 1]);
        }
        __syncwarp();
      };
      auto state = [&](int it) {  // dS^T
        const int st = ring.st, wb = it % C::wv_bufs, db = it % C::ds_bufs;
        const uint32_t kd = desc_lo(sb + L::k + st * NK * kBox, kBox);
        if (it >= C::ds_bufs) ok &= wait_for(&m.ds_free[db], (it / C::ds_bufs - 1) & 1);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          ok &= wait_for(&m.wv_ready[wb][half], (it / C::wv_bufs) & 1);
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int part = 2; part >= 0; --part)  // the small parts first
#pragma unroll
              for (int kk = 0; kk < 2; ++kk)
                umma_ts(tm + C::ds + 64 * NK * db, tm + C::wv + 96 * wb + 32 * part + 16 * half + 8 * kk,
                        desc_of(kd + (half * 4096u + kk * 2048u >> 4)), idesc_bf16(128, 64 * NK, false, true),
                        half > 0 || part < 2 || kk > 0);
            umma_commit(&m.wv_free[wb][half]);
            if (half == 1) umma_commit(&m.ds_full[db]);
            if (half == 1) umma_commit(&m.empty[st]);
          }
          __syncwarp();
        }
      };
#pragma unroll 1
      for (int it = 0; it < n_chunks && !bad; ++it, ring.next()) {
        if (FULL) scores(it);
        state(it);
        bad = __any_sync(0xffffffffu, !ok);
      }
      bad |= !drain(0);
    } else if (FULL && warp == kOutMmaWarp) {
      // ---- the output's products ------------------------------------------------------
      Ring<kStages> ring;
      bool ok = true;
      auto inter = [&](int it) {  // OI^T
        const int st = ring.st;
        ok &= wait_for(&m.full[st], ring.ph);
        ok &= wait_for(&m.s_ready, it & 1);
        if (it > 0) ok &= wait_for(&m.oi_free, (it - 1) & 1);
        tc_fence_after();
        const uint32_t qd = desc_lo(sb + L::q + st * NK * kBox, 0);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4 * NK; ++kk)
            umma_ts(tm + C::oi, tm + C::s + 8 * kk, desc_of(qd + (((kk >> 2) * kBox + (kk & 3) * 32u) >> 4)),
                    idesc_bf16(128, 64, false, false), kk > 0);
          umma_commit(&m.s_free);
        }
        __syncwarp();
      };
      auto within = [&](int it) {  // OP^T
        const int st = ring.st;
        ok &= wait_for(&m.p_ready[it & 1], (it >> 1) & 1);
        tc_fence_after();
        // Wide: both tiles of v. Head x of a pair: its tile and the zero tile, in the order of the blocks.
        const uint32_t step = WIDE ? kBox : (st + 1) * kBox;
        const uint32_t v0 = desc_lo(sb + L::va(st), step), v1 = desc_lo(sb + L::zero, step);
        const uint32_t pd = desc_lo(sb + L::ptile(it, 0), 0);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_f16(tm + C::x + 64 * (it & 1), desc_of(v0 + (kk * 2048u >> 4)), desc_of(pd + (kk * 32u >> 4)),
                     idesc_bf16(128, 64, true, false), kk > 0);
          if (!WIDE && u.nheads == 2) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_f16(tm + C::x + 64 * (it & 1), desc_of(v1 + (kk * 2048u >> 4)), desc_of(pd + ((kBox + kk * 32u) >> 4)),
                       idesc_bf16(128, 64, true, false), 1);
          }
          umma_commit(&m.o_full[it & 1]);
          umma_commit(&m.empty[st]);
        }
        __syncwarp();
      };
#pragma unroll 1
      for (int it = 0; it < n_chunks && !bad; ++it, ring.next()) {
        inter(it);
        within(it);
        bad = __any_sync(0xffffffffu, !ok);
      }
      bad |= !drain(1);
    } else if (warp == kSumWarp) {
      // ---- decay sums -------------------------------------------------------------------
      const int x = lane / kLanes, tok = lane % kLanes * kT;
      const bool mine = x < u.nheads;
      float seg_total = 0.f;
      // This lane's decays of the chunk that is loaded next, and how many are before the length.
      const float* ahead = l.decay + u.b * l.sg[0] + (u.head0 + x) * l.sg[1] + (u.first * kC + tok) * l.sg[2];
      int left = mine ? u.len - u.first * kC - tok : 0;
#pragma unroll 1
      for (int it = 0; it < n_chunks; ++it) {
        const int sl = it % kSums, live = u.live(it);
        float c[kT], after[kT];
#pragma unroll
        for (int j = 0; j < kT; ++j) {
          const float a = decays[j] * kLog2e;
          c[j] = a < kMinLog2 ? kMinLog2 : a;  // NaN stays
        }
        float was[kT];
#pragma unroll
        for (int j = 0; j < kT; ++j) was[j] = decays[j];
        ahead += kC * l.sg[2], left -= kC;
        if (it + 1 < n_chunks) {
#pragma unroll
          for (int j = 0; j < kT; ++j) decays[j] = j < left ? ahead[j * l.sg[2]] : 0.f;
        }
        // Sums up to each token, and of those after it, without subtracting large sums.
        after[kT - 1] = 0.f;
#pragma unroll
        for (int j = kT - 2; j >= 0; --j) after[j] = after[j + 1] + c[j + 1];
        float r = after[0] + c[0];
#pragma unroll
        for (int j = 1; j < kT; ++j) c[j] += c[j - 1];
        float f = c[kT - 1];
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) {
          const float a = __shfl_up_sync(0xffffffffu, f, o, kLanes), b = __shfl_down_sync(0xffffffffu, r, o, kLanes);
          if (lane % kLanes >= o) f += a;
          if (lane % kLanes + o < kLanes) r += b;
        }
        float before = __shfl_up_sync(0xffffffffu, f, 1, kLanes), behind = __shfl_down_sync(0xffffffffu, r, 1, kLanes);
        const float total = __shfl_sync(0xffffffffu, r, 0, kLanes), mid = 0.5f * total;
        if (lane % kLanes == 0) before = 0.f;
        if (lane % kLanes == kLanes - 1) behind = 0.f;
        // e^{c_i - c_j} as a product of two factors, where none leaves 2^+-120 (the scale's part: 2^+-20).
        bool near = l.scale >= 0x1p-20f && l.scale <= 0x1p20f;
#pragma unroll
        for (int j = 0; j < kT; ++j) {
          c[j] += before;
          after[j] += behind;
          near = near && fabsf(c[j] - mid) <= 100.f;
        }
        const uint32_t votes = __ballot_sync(0xffffffffu, near);
        const bool factors = WIDE ? votes == 0xffffffffu : (votes >> (16 * x) & 0xffffu) == 0xffffu;
        bad |= it >= kSums && !wait_for(&m.sums_free[sl], (it / kSums - 1) & 1);
        if (__any_sync(0xffffffffu, bad)) {
          bad = true;
          break;
        }
#pragma unroll
        for (int j = 0; j < kT; j += 2) {
          auto put = [&](float* to, float a, float b) { *reinterpret_cast<float2*>(to + tok + j) = make_float2(a, b); };
          const float c0 = c[j], c1 = c[j + 1];
          put(m.row[sl][x], factors ? l.scale * ex2_approx(c0 - mid) : c0, factors ? l.scale * ex2_approx(c1 - mid) : c1);
          put(m.col[sl][x], factors ? ex2_approx(mid - c0) : -c0, factors ? ex2_approx(mid - c1) : -c1);
          put(m.ecs[sl][x], l.scale * ex2_approx(c0), l.scale * ex2_approx(c1));
          put(m.w[sl][x], tok + j < live ? ex2_approx(after[j]) : 0.f, tok + j + 1 < live ? ex2_approx(after[j + 1]) : 0.f);
        }
        if (lane % kLanes == 0) {
          const float e = ex2_approx(total);
          m.total[sl][x] = e == 0.f ? kTiny : e;
          m.factors[sl][x] = factors;
        }
        seg_total += total;
        // A decay of -inf, after which nothing of the state before may be left, also where that is not
        // finite. (Such a chunk's sum is kMinLog2 or less.)
        if (__builtin_expect(__any_sync(0xffffffffu, total <= kMinLog2), 0)) {
          int reset = kC;
#pragma unroll
          for (int j = kT - 1; j >= 0; --j) reset = was[j] == -INFINITY ? tok + j : reset;
#pragma unroll 1
          for (int o = 1; o < kLanes; o <<= 1) reset = min(reset, __shfl_xor_sync(0xffffffffu, reset, o, kLanes));
          if (reset < kC) {
            if (lane % kLanes == 0) m.total[sl][x] = -1.f, m.reset[sl][x] = reset;
            seg_total = -INFINITY;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.sums[sl]);
      }
      if (!FULL && mine && lane % kLanes == 0 && !bad)
        p.seg_decay[(static_cast<int64_t>(u.b) * l.H + u.head0 + x) * p.segs + u.seg] = seg_total;
    }
    __syncwarp();
  } else if (warp >= kOutWarp) {
    // ---- outputs ------------------------------------------------------------------------
    fewer_registers<R::out>();
    if (FULL) {
      const Unit u = m.unit;
      const int n_chunks = u.last - u.first;
      const int half = (warp - kOutWarp) >> 2;  // 32 tokens
      const int hd = WIDE ? 0 : q4 >> 1, head = u.head0 + hd;
      const int ocol = WIDE ? 32 * q4 : 32 * (q4 & 1);
      const bool stores = ocol < l.P && hd < u.nheads;
      const uint32_t stage = sb + L::o + (warp - kOutWarp) * 2048u;  // 32 tokens x 32 columns
      fill_rows(p, u, u.last * kC, tid - 32 * kOutWarp, 256, 0u);  // chunks past the length
      for (int it = 0; it < n_chunks; ++it) {
        const int sl = it % kSums, t0 = (u.first + it) * kC + 32 * half;
        bad |= !wait_for(&m.sums[sl], (it / kSums) & 1);
        const bool resets = m.total[sl][hd < u.nheads ? hd : 0] < 0.f;
        bad |= !wait_for(&m.o_full[it & 1], (it >> 1) & 1);
        tc_fence_after();
        if (__any_sync(0xffffffffu, bad || resets)) {
          if (__any_sync(0xffffffffu, bad)) {
            bad = true;
            break;
          }
          // From a decay of -inf on, tokens have nothing of the state: their columns of OI are zero, also
          // where the state is not finite.
#pragma unroll 1
          for (int t = max(m.reset[sl][hd < u.nheads ? hd : 0] - 32 * half, 0); t < 32; ++t)
            tmem_st1(tm + C::oi + 32 * half + t + tl, 0u);
          tmem_wait_st();
        }
        if (lane == 0) tma_store_wait_read();
        __syncwarp();
        const float* ecs = &m.ecs[sl][hd < u.nheads ? hd : 0][32 * half + 2 * (lane & 3)];
        const uint32_t from = tm + 32 * half + tl;
        const int live = u.live(it);
        // All of q S first, whose columns the next chunk waits for: [16 tokens][16 lanes].
        float oi[4][8];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld_frag2(from + C::oi + 16 * (i >> 1) + (16u * (i & 1) << 16), oi[i]);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.oi_free);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int x = i >> 1, sub = i & 1;
          float op[8];
          tmem_ld_frag2(from + C::x + 64 * (it & 1) + 16 * x + (16u * sub << 16), op);
          const float2 e[2] = {*reinterpret_cast<const float2*>(ecs + 16 * x),
                               *reinterpret_cast<const float2*>(ecs + 16 * x + 8)};
          tmem_wait_ld();
          uint32_t o[4];  // [token group y][row group]: tokens 8 y + 2 (lane % 4) + {0, 1}
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 y = fma2(make_float2(oi[i][2 * j], oi[i][2 * j + 1]), e[j >> 1], make_float2(op[2 * j], op[2 * j + 1]));
            o[j] = pack_bf16x2(y.x, y.y);
          }
          if (live < kC) {  // rows past the length are zero
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int left = live - 32 * half - 2 * (lane & 3) - 16 * x - 8 * (j >> 1);
              o[j] &= left > 1 ? 0xffffffffu : left > 0 ? 0xffffu : 0u;
            }
          }
          stsm_x4_t(stage + x * 1024u + (lane >> 4) * 512u + (lane & 7) * 64u +
                        (((2 * sub + ((lane >> 3) & 1)) ^ ((lane >> 1) & 3)) << 4),
                    o[0], o[1], o[2], o[3]);
        }
        tc_fence_before();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&m.op_free[it & 1]);
          mbar_arrive(&m.sums_free[sl]);
          if (stores && t0 < l.T) tma_store_4d(&p.tm_o, stage, ocol, head, t0, u.b);
        }
      }
      if (lane == 0) tma_store_wait_read();
      __syncwarp();
    }
  } else if (warp >= kScoreWarp) {
    // ---- scores to weights: P = D e^{c_i - c_j} for j <= i ------------------------------
    fewer_registers<R::score>();
    if (FULL) {
      const Unit u = m.unit;
      const int n_chunks = u.last - u.first;
      const int half = (warp - kScoreWarp) >> 2;  // 32 columns
      // Rows i0 and i0 + 8; 16 columns at a time: j0 + 16 z + 8 y + {0, 1}, y < 2. Columns past
      // the warp's last row are left alone.
      const int i0 = 16 * q4 + (lane >> 2), j0 = 32 * half + 2 * (lane & 3);
      const int steps = min(2, max(0, q4 + 1 - 2 * half));
      const int heads = WIDE ? 1 : u.nheads;
      // The zero tile, and P's tiles: what lies above the diagonal is never written.
      for (int i = tid - 32 * kScoreWarp; i < (WIDE ? 2 : 4) * kBox / 16; i += 256)
        sts16(sb + L::p + 16 * i, make_uint4(0, 0, 0, 0));
      if (!WIDE)
        for (int i = tid - 32 * kScoreWarp; i < kBox / 16; i += 256) sts16(sb + L::zero + 16 * i, make_uint4(0, 0, 0, 0));
      bad = bar_or(3, 256, false);
      // Pairs of the last step that lie on or below the diagonal, [y][row group].
      uint32_t keep[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int left = i0 + 8 * (j & 1) - (j0 + 16 * (q4 - 2 * half) + 8 * (j >> 1));
        keep[j] = left >= 1 ? 0xffffffffu : left == 0 ? 0xffffu : 0u;
      }
      Ring<kStages> ring;
      for (int it = 0; it < n_chunks; ++it, ring.next()) {
        const int sl = it % kSums;
        bad |= !wait_for(&m.sums[sl], (it / kSums) & 1);
        bad |= it >= 2 && !wait_for(&m.o_full[it & 1], ((it >> 1) - 1) & 1);  // P's tiles have been read
        bad |= !wait_for(&m.d_full[it & 1], (it >> 1) & 1);
        tc_fence_after();
        if (__any_sync(0xffffffffu, bad)) {
          bad = true;
          break;
        }
        const int live = u.live(it);
        if (live < kC) {  // as the prepared values: rows past the length are zero before v is an operand
          const int st = ring.st, vecs = (kC - live) * 8;
          for (int i = tid - 32 * kScoreWarp; i < (WIDE || u.nheads == 2 ? 2 : 1) * vecs; i += 256)
            sts16(sb + (i < vecs ? L::va(st) : L::vb(st)) + live * 128 + 16 * (i % vecs), make_uint4(0, 0, 0, 0));
        }
#pragma unroll 1
        for (int z = 0; z < steps; ++z) {
          float d[8];
          tmem_ld_frag2(tm + C::x + 64 * (it & 1) + 32 * half + 16 * z + tl, d);
          tmem_wait_ld();
          const bool diagonal = 2 * half + z == q4;
#pragma unroll 1
          for (int x = 0; x < heads; ++x) {
            const float r[2] = {m.row[sl][x][i0], m.row[sl][x][i0 + 8]};
            const float* cj = m.col[sl][x] + j0 + 16 * z;
            const float2 c[2] = {*reinterpret_cast<const float2*>(cj), *reinterpret_cast<const float2*>(cj + 8)};
            uint32_t o[4];  // [y][row group]
            if (m.factors[sl][x]) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 e = mul2(make_float2(r[j & 1], r[j & 1]), c[j >> 1]);
                const float2 w = mul2(e, make_float2(d[2 * j], d[2 * j + 1]));
                o[j] = pack_bf16x2(w.x, w.y);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                o[j] = pack_bf16x2(l.scale * ex2_approx(r[j & 1] + c[j >> 1].x) * d[2 * j],
                                   l.scale * ex2_approx(r[j & 1] + c[j >> 1].y) * d[2 * j + 1]);
            }
            if (diagonal) {
#pragma unroll
              for (int j = 0; j < 4; ++j) o[j] &= keep[j];
            }
            const uint32_t ps = sb + L::ptile(it, x) + i0 * 128u + 4 * (lane & 3);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint32_t to = ps + (((4 * half + 2 * z + y) ^ (lane >> 2)) << 4);
              sts4(to, o[2 * y]);
              sts4(to + 1024u, o[2 * y + 1]);
            }
          }
        }
        tc_fence_before();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.p_ready[it & 1]);
      }
    }
  } else if (warp >= kPrepWarp) {
    // ---- weighted values, transposed into TMEM -------------------------------------------
    fewer_registers<R::prep>();
    const Unit u = m.unit;
    const int n_chunks = u.last - u.first;
    const bool two = WIDE || u.nheads == 2;
    const int pt = tid - 32 * kPrepWarp, half = (warp - kPrepWarp) >> 2;  // 32 tokens
    const int blk = q4 >> 1;                       // block of value columns of this warp's lanes
    const int hd = WIDE ? 0 : blk;
    const bool mine = blk == 0 || two;
    if (!mine) {  // lanes without values stay zero
      const uint32_t z[16] = {};
      for (int i = 0; i < 3 * C::wv_bufs; ++i) tmem_st16(tm + C::wv + 32 * i + 16 * half + tl, z);
    }
    Ring<kStages> ring;
    bool met = u.live(n_chunks - 1) == kC;  // at the barrier of a partial last chunk, if there is one
    for (int it = 0; it < n_chunks; ++it, ring.next()) {
      const int st = ring.st, sl = it % kSums, live = u.live(it), wb = it % C::wv_bufs;
      bad |= !wait_for(&m.full[st], ring.ph);
      bad |= !wait_for(&m.sums[sl], (it / kSums) & 1);
      if (live < kC) {
        // Rows past the length hold anything: as operands they must be zero. (The scores may
        // read k before or after: those columns are masked.)
        const int vecs = (kC - live) * 8;
        for (int i = pt; i < (NK + (two ? 2 : 1)) * vecs; i += 256) {
          const int box = i / vecs, at = i % vecs;
          const uint32_t base = box < NK ? L::k + (st * NK + box) * kBox : box == NK ? L::va(st) : L::vb(st);
          sts16(sb + base + live * 128 + 16 * at, make_uint4(0, 0, 0, 0));
        }
        fence_async_smem();
        bad = bar_or(2, 256, bad);
        met = true;
      }
      if (__any_sync(0xffffffffu, bad)) {
        bad = true;
        break;
      }
      // The operand is free once the state product before has read it.
      if (it >= C::wv_bufs) bad |= !wait_for(&m.wv_free[wb][half], (it / C::wv_bufs - 1) & 1);
      tc_fence_after();
      if (mine) {
        const float* w = &m.w[sl][hd][32 * half + 2 * (lane & 3)];
        const uint32_t src = sb + (blk ? L::vb(st) : L::va(st)) + half * 4096u + (lane >> 4) * 1024u + (lane & 7) * 128u;
        const uint32_t chunk = (4 * (q4 & 1) + ((lane >> 3) & 1)) ^ (lane & 7);
#pragma unroll 2
        for (int i = 0; i < 4; ++i) {  // 16 lanes (sub) x 16 tokens
          const int sub = i & 1, x = i >> 1;
          uint32_t in[4], hi[4], mid[4], lo[4];
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                       : "=r"(in[0]), "=r"(in[1]), "=r"(in[2]), "=r"(in[3])
                       : "r"(src + x * 2048u + ((chunk ^ (2 * sub)) << 4))
                       : "memory");
          const float2 wj[2] = {*reinterpret_cast<const float2*>(w + 16 * x),
                                *reinterpret_cast<const float2*>(w + 16 * x + 8)};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float2 y = mul2(make_float2(__uint_as_float(in[j] << 16), __uint_as_float(in[j] & 0xffff0000u)), wj[j >> 1]);
            hi[j] = take_bf16(y);
            mid[j] = take_bf16(y);
            lo[j] = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x7632);
          }
          const uint32_t to = tm + C::wv + 96 * wb + 16 * half + 8 * x + tl + (16u * sub << 16);
          tmem_st_16x128_x2(to, hi);
          tmem_st_16x128_x2(to + 32, mid);
          tmem_st_16x128_x2(to + 64, lo);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.wv_ready[wb][half]);
    }
    if (!met) bar_or(2, 256, true);
  } else {
    // ---- state ------------------------------------------------------------------------------
    more_registers<R::state>();
    const Unit u = m.unit;
    const int n_chunks = u.last - u.first;
    const int row = 32 * q4 + lane;              // accumulator lane
    const int blk = row >> 6;                    // block of value columns
    const int hd = WIDE ? 0 : blk;               // head of the CTA
    const int col = WIDE ? row : row & 63;       // value column in the head
    const bool on = col < l.P && hd < u.nheads;
    constexpr int kNS = 64 * NK;                 // state values of a thread: the key columns of a value
    // States go between shared memory and registers through TMEM, 16 columns at a time: a loop
    // over rows can address TMEM, not registers, and unrolled it would be 20 KB of code that
    // every CTA has to fetch. This lane's value of the first of those rows, in two areas:
    auto rows_at = [&](uint32_t a0, uint32_t a1, int n) {
      return sb + (WIDE ? (n < 64 ? a0 : a1) + static_cast<uint32_t>((n & 63) * l.P) * 4 : (blk ? a1 : a0) + n * l.P * 4) +
             col * 4;
    };
    float s[kNS];
    if (!has_init) {
#pragma unroll
      for (int i = 0; i < kNS; ++i) s[i] = 0.f;
    } else {
      bad |= !wait_for(&m.init_full, 0);
      // Columns that nothing uses before the state is there: the second chunk's D, and OI.
      auto columns = [&](int n) { return tm + (n < 64 ? C::x + 64 + n : C::oi + n - 64) + tl; };
#pragma unroll 1
      for (int n = 0; n < kNS; n += 16) {
        uint32_t r[16], from = rows_at(L::init0, L::init1, n);
#pragma unroll
        for (int j = 0; j < 16; ++j, from += l.P * 4) {
          r[j] = 0;
          if (on && n + j < l.N) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r[j]) : "r"(from) : "memory");
        }
        tmem_st16(columns(n), r);
      }
      tmem_wait_st();
#pragma unroll
      for (int n = 0; n < kNS; n += 16) tmem_ld16(columns(n), *reinterpret_cast<float(*)[16]>(s + n));
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.init_read);
    }
    // The state rounded to BF16, as the operand of q S.
    auto put_state = [&]() {
#pragma unroll
      for (int i = 0; i < kNS; i += 16) {
        uint32_t r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = pack_bf16x2(s[i + 2 * j], s[i + 2 * j + 1]);
        tmem_st8(tm + C::s + i / 2 + tl, r);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.s_ready);
    };
    if (FULL) put_state();
    for (int it = 0; it < n_chunks; ++it) {
      const int sl = it % kSums, db = it % C::ds_bufs;
      // S = e^{c_C} S + dS.
      bad |= !wait_for(&m.sums[sl], (it / kSums) & 1);
      float a = m.total[sl][hd < u.nheads ? hd : 0];
      bad |= !wait_for(&m.ds_full[db], (it / C::ds_bufs) & 1);
      tc_fence_after();
      if (__any_sync(0xffffffffu, bad)) {
        bad = true;
        break;
      }
      if (__builtin_expect(a < 0.f, 0)) {  // a decay of -inf: nothing of S, also where it is not finite
#pragma unroll
        for (int i = 0; i < kNS; i += 16)  // (in its place something finite, in few instructions)
          tmem_ld16(tm + C::ds + 64 * NK * db + i + tl, *reinterpret_cast<float(*)[16]>(s + i));
        tmem_wait_ld();
        a = 0.f;
      }
      constexpr int kBatch = NK == 1 ? 32 : 16;  // columns on their way at a time, as registers allow
#pragma unroll
      for (int i = 0; i < kNS; i += kBatch) {
        float d[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; j += 16)
          tmem_ld16(tm + C::ds + 64 * NK * db + i + j + tl, *reinterpret_cast<float(*)[16]>(d + j));
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < kBatch; j += 2) {
          const float2 x = fma2(make_float2(a, a), make_float2(s[i + j], s[i + j + 1]), make_float2(d[j], d[j + 1]));
          s[i + j] = x.x;
          s[i + j + 1] = x.y;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&m.ds_free[db]);
        mbar_arrive(&m.sums_free[sl]);
      }
      if (FULL && it + 1 < n_chunks) {
        bad |= !wait_for(&m.s_free, it & 1);  // the operand has been read
        tc_fence_after();
        if (__any_sync(0xffffffffu, bad)) {
          bad = true;
          break;
        }
        put_state();
      }
    }
    // The state after the last chunk, through shared memory: every tile there has been read.
    if (FULL) bad |= !wait_for(&m.o_full[(n_chunks - 1) & 1], ((n_chunks - 1) >> 1) & 1);
    if (!FULL || (u.ends_row() && l.state)) {
#pragma unroll
      for (int n = 0; n < kNS; n += 8) {
        uint32_t r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = __float_as_uint(s[n + j]);
        tmem_st8(tm + C::ds + n + tl, r);
      }
      tmem_wait_st();
#pragma unroll 1
      for (int n = 0; n < kNS; n += 16) {
        float r[16];
        tmem_ld16(tm + C::ds + n + tl, r);
        tmem_wait_ld();
        uint32_t to = rows_at(L::last0, L::last1, n);
#pragma unroll
        for (int j = 0; j < 16; ++j, to += l.P * 4)
          if (on && n + j < l.N) sts4(to, __float_as_uint(r[j]));
      }
      fence_async_smem();
      bad = bar_or(1, 128, bad);
      if (tid == 0 && !bad) {
        for (int x = 0; x < pieces(u); ++x)
          bulk_store(FULL ? pool_piece(u, x) : seg_piece(u, u.seg + 1, x), sb + (x ? L::last1 : L::last0), piece_bytes(x));
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        tma_store_wait_read();
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  const bool any = __syncthreads_or(bad);
  if (any && tid == 0) {
    atomicExch(&g_linear_error, kLinearGaveUp);
    if (p.err_host) {
      *reinterpret_cast<volatile int*>(p.err_host) = kLinearGaveUp;
      __threadfence_system();
    }
  }
  if (warp == kStateMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tm, 512);
  }
}

// The state before every segment, from the segments' own states: S_in(0) = the carried
// state, S_in(i + 1) = 2^decay(i) S_in(i) + own(i). Thread: four neighbouring values of
// one head; own(i) lies where S_in(i + 1) goes.
__global__ void __launch_bounds__(256) linear_join_kernel(const __grid_constant__ ChunkParams p) {
  const LinearParams& l = p.l;
  const int quads = l.N * l.P / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<int64_t>(l.B) * l.H * quads) return;
  const int64_t row = i / quads;
  const int e = static_cast<int>(i % quads) * 4;
  const int b = static_cast<int>(row / l.H), h = static_cast<int>(row % l.H);
  int64_t len = l.T;
  if (l.lengths) len = min(max(l.lengths[b], static_cast<int64_t>(0)), len);
  const int live = static_cast<int>((len + kC - 1) / kC);
  const int segs = (live + p.seg_chunks - 1) / p.seg_chunks;
  if (segs == 0) return;
  float* own = p.seg_state + row * p.segs * l.N * l.P + e;
  const int64_t step = static_cast<int64_t>(l.N) * l.P;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  const int64_t slot = l.slots ? l.slots[b] : b;
  if (!l.fresh && l.state && slot >= 0 && slot < l.nslots)
    s = *reinterpret_cast<const float4*>(l.state + slot * l.ss[0] + h * l.ss[1] + e);
  *reinterpret_cast<float4*>(own) = s;
#pragma unroll 4
  for (int g = 1; g < segs; ++g) {
    const float total = p.seg_decay[row * p.segs + g - 1], e = ex2_approx(total), a = e == 0.f ? kTiny : e;
    if (total == -INFINITY) s = make_float4(0.f, 0.f, 0.f, 0.f);  // a decay of -inf in the segment
    const float4 d = __ldcg(reinterpret_cast<const float4*>(own + g * step));
    s.x = fmaf(a, s.x, d.x);
    s.y = fmaf(a, s.y, d.y);
    s.z = fmaf(a, s.z, d.z);
    s.w = fmaf(a, s.w, d.w);
    *reinterpret_cast<float4*>(own + g * step) = s;
  }
}

// ---- host side ---------------------------------------------------------------------
// The driver's encoder of tensor maps, looked up once (also where several threads call first).
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const auto fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// [B, T, heads, width] BF16 rows as a map with boxes of `side` tokens x `side` columns of one
// head, swizzled over a row of the box; columns past the width and tokens past T read as
// zero and are not written.
bool encode(CUtensorMap* map, const void* base, int width, int heads, int T, int B, const int64_t* s,
            unsigned side = 64) {
  const int64_t st[3] = {s[2], s[1], s[0]};
  const int ext[3] = {heads, T, B};
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(T),
                              static_cast<cuuint64_t>(B)};
  cuuint64_t strides[3];
  if (reinterpret_cast<uintptr_t>(base) % 16) return false;
  for (int i = 0; i < 3; ++i) {
    const int64_t bytes = ext[i] == 1 ? (width * 2 + 15) / 16 * 16 : st[i] * 2;  // a lone entry's stride is never used
    if (bytes <= 0 || bytes % 16 || bytes >= (1ll << 40)) return false;
    strides[i] = static_cast<cuuint64_t>(bytes);
  }
  const cuuint32_t box[4] = {side, 1, side, 1}, one[4] = {1, 1, 1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, one,
                  CU_TENSOR_MAP_INTERLEAVE_NONE,
                  side == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
  int pairs, chunks, segs, seg_chunks;
  int64_t rows, state_bytes, bytes;
};

// A prompt shorter than this runs token by token, in batches of eight tokens. With a carried state, us
// token by token / in a chunk:
//   N 128, P 64, 1 row of 12 heads, 16 of 12, 32 of 32
//     12 tokens    6.8 / 9.6    11.3 / 10.1   41.0 / 37.8
//     16           6.8 / 9.6    11.5 / 10.1   41.7 / 37.5
//     17           8.2 / 9.6    14.5 / 10.0   53.9 / 37.5
//   N 64, P 64, 1, 16 and 80 rows of 8 heads
//     16           5.3 / 7.9     6.7 / 8.1    19.2 / 22.8
//     17           6.4 / 7.8     8.1 / 8.1    24.4 / 22.8
constexpr int kMinTokens = 17;

bool plan_of(int B, int T, int H, int Hq, int N, int P, int dtype, Plan& x) {
  if (dtype != TF_BF16 || N > 128 || P > 128 || T < kMinTokens) return false;
  const int share = H / Hq;
  x.pairs = P > 64 ? share : (share + 1) / 2;
  x.chunks = (T + kC - 1) / kC;
  x.rows = static_cast<int64_t>(B) * Hq * x.pairs;
  // As many segments as there are SMs for, of four chunks or more. Each is worked on twice, and the join
  // and the further launches take as long as six chunks; where that is no gain, rows stay whole.
  // 12 heads, N 128, P 64 (six CTAs a row), us cut / whole:
  //   1 x 512, 1024, 3600 tokens     25.9 / 19.1   27.0 / 30.4   29.6 / 87.8
  //   6 x 512, 1024, 3600            28.1 / 19.5   30.9 / 30.8   55.4 / 89.1
  //   10 x 512, 1024, 3600           30.4 / 19.9   39.6 / 31.0   88.8 / 89.3
  //   12 x 512, 1024, 3600           31.3 / 20.2   40.6 / 31.3   91.1 / 89.6
  const int64_t most = std::min<int64_t>(sm_count() / x.rows, (x.chunks + 3) / 4);
  x.seg_chunks = x.chunks;
  if (most > 1) {
    const int part = static_cast<int>((x.chunks + most - 1) / most);
    if (2 * part + 6 < x.chunks) x.seg_chunks = part;
  }
  x.segs = (x.chunks + x.seg_chunks - 1) / x.seg_chunks;
  x.state_bytes = x.segs > 1 ? static_cast<int64_t>(B) * H * x.segs * N * P * 4 : 0;
  x.bytes = x.state_bytes + (x.segs > 1 ? static_cast<int64_t>(B) * H * x.segs * 4 : 0);
  return true;
}

template <int NK, bool WIDE, bool FULL>
void launch_chunks(const ChunkParams& p, unsigned grid, cudaStream_t stream) {
  auto kernel = linear_chunk_kernel<NK, WIDE, FULL>;
  constexpr int bytes = Layout<NK, WIDE, FULL>::bytes;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel has its shared memory size
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(ready.load() >> dev & 1)) {
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    ready.fetch_or(1ull << dev);
  }
  kernel<<<grid, kThreads, bytes, stream>>>(p);
}
template <bool FULL>
void launch_any(const ChunkParams& p, unsigned grid, cudaStream_t stream) {
  if (p.l.N > 64) {
    if (p.l.P > 64) launch_chunks<2, true, FULL>(p, grid, stream);
    else launch_chunks<2, false, FULL>(p, grid, stream);
  } else {
    if (p.l.P > 64) launch_chunks<1, true, FULL>(p, grid, stream);
    else launch_chunks<1, false, FULL>(p, grid, stream);
  }
}

}  // namespace

int64_t linear_chunk_workspace(int B, int T, int H, int Hq, int N, int P, int dtype) {
  Plan x;
  return plan_of(B, T, H, Hq, N, P, dtype, x) ? x.bytes : -1;
}

int launch_linear_chunks(const LinearParams& l, int dtype, void* workspace, int64_t workspace_bytes,
                         cudaStream_t stream) {
  Plan x;
  if (!plan_of(l.B, l.T, l.H, l.Hq, l.N, l.P, dtype, x) || !encoder()) return -1;
  ChunkParams p{};
  if (!encode(&p.tm_q, l.q, l.N, l.Hq, l.T, l.B, l.sq) || !encode(&p.tm_k, l.k, l.N, l.Hq, l.T, l.B, l.sk) ||
      !encode(&p.tm_v, l.v, l.P, l.H, l.T, l.B, l.sv) || !encode(&p.tm_o, l.out, l.P, l.H, l.T, l.B, l.so, 32))
    return -1;
  if (x.rows * x.segs > 0x7fffffffll) return TF_ERR_SIZE;
  if (x.bytes > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256)) return TF_ERR_ARG;
  if (workspace_bytes < x.bytes) return TF_ERR_SIZE;
  p.l = l;
  p.pairs = x.pairs, p.segs = x.segs, p.seg_chunks = x.seg_chunks;
  p.seg_state = static_cast<float*>(workspace);
  p.seg_decay = reinterpret_cast<float*>(static_cast<char*>(workspace) + x.state_bytes);
  p.err_host = host_error_word();
  p.tries = static_cast<uint32_t>(std::min(flag_wait_limit_ns() / kTryNs, 0xffffffffull));
  const unsigned grid = static_cast<unsigned>(x.rows * x.segs);
  if (x.segs > 1) {
    launch_any<false>(p, grid, stream);
    const int64_t quads = static_cast<int64_t>(l.B) * l.H * l.N * l.P / 4;
    linear_join_kernel<<<static_cast<unsigned>((quads + 255) / 256), 256, 0, stream>>>(p);
  }
  launch_any<true>(p, grid, stream);
  return launch_status();
}

int read_linear_error(int reset) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_linear_error, sizeof(int));
  if (reset) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_linear_error, &zero, sizeof(int));
  }
  return v;
}

}  // namespace tf
