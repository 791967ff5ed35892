// Attention of drafted trees, chains or single tokens over a paged KV cache:
//   out_i = sum_j p_ij v_j,  p_ij = exp(s_ij - m_i) / sum_j exp(s_ij - m_i),
//   s_ij = scale q_i . k_j over the keys j that row i sees:
// all rows of the cache in front of the request's new tokens, and of the new
// tokens' own rows those that its mask names (or j <= i without a mask).
//
// The query heads that share a KV head are rows of one tile: row r of a tile is
// token r / G, head r % G (G = Hq / Hkv), so K and V are read once for all of them
// and a tile of 128 rows holds 128 / G tokens.  A work item is (request, KV head,
// one tile of tokens); its keys come in tiles of 64.
//
// Two persistent CTAs per SM, each warp-specialised:
//   warps 0-3  softmax, one thread per row
//   warp 4     walks this CTA's share of the work and hands out its items; TMA: an
//              item's Q, and the pages of a K or V tile into a ring of stages, one lane
//              per box, 128-byte swizzle
//   warp 5     tcgen05.mma: S = Q K^T (128 x 64, both operands from shared
//              memory), O += P V (P from tensor memory)
// Tensor memory: two buffers of scores (64 columns each; P is written over the
// scores it comes from) and O (D columns).  While the softmax has one tile of scores
// the tensor core computes the next one into the other buffer.  The two CTAs
// of an SM hide each other's waits: while one is between two items (its last product,
// the output, the next Q) the other keeps the memory and the tensor core busy.
//
// Work is split evenly over the CTAs: every CTA adds up the key tiles of all items
// (from the lengths, on the GPU; an item counts kItemUnits more for its fixed cost) and
// takes its share of the line, which may begin and end inside an item.  There are two
// such lines.  On the first lie the pairs of query tiles that read the same keys: two CTAs
// take a share of it together, one tile each, so the second reading finds the
// keys in L2 (one tile behind the other, a whole pass over the cache lay between the two
// readings: 32 trees of 64 tokens over 4096 took 130 us so, and 109 in pairs).  On the second lie the
// single tiles.  An item that lies in several CTAs is written as unnormalised fp32 partials
// with their maxima and sums, which a second small kernel joins in a fixed order.
//
// The running maximum is only raised (and O rescaled) when it grows by more than
// 8 in base 2: the probabilities then stay below 2^8 (fp16 keeps them 2^7 times as large,
// see kLift), the sums are fp32, and nearly all tiles leave O alone.  S, maxima, sums and O are fp32; P is
// rounded to the activation type, as the tensor core takes no other operand.
//
// Masked keys contribute nothing, whatever they hold: masked scores are replaced,
// not added to, and because 0 * inf is not 0 the rows of V beyond the request's
// end are zeroed in shared memory, and values that are not finite in rows that
// some query does not see are zeroed there and added back, in the epilogue, to the
// rows that do see them.  Only tiles that hold such keys pay for this.
//
// Bound: HBM for single tokens, where every K and V row is used by G rows only; the tensor
// core and the softmax for many rows.  The twelve products of a tile (Q K^T 8 of 61 cycles, as 64 keys
// re-read all of Q; P V 4 of 65) take 748 cycles alone, 512 of them arithmetic; a tile of 128 x 64
// takes an SM 1011 cycles (prompts below, by their time and clock).
// 32 query heads, 8 KV heads of 128, bf16, on a B200, calls of a CUDA graph of a few milliseconds,
// with the mean SM clock (of 1965 MHz; the power limit sets it), and after a second of them:
//   64 single tokens, up to 8192 rows   207 us at 1831 MHz  6.4 TB/s                213 us
//   32 trees of up to 64, 4096 rows     107 us at 1660 MHz  3.4 TB/s, 600 TFLOP/s   124 us
//   3 x up to 2048 tokens, 4096 rows    349 us at 1685 MHz  1010 TFLOP/s            400 us
//   1000 single tokens, up to 500 rows  214 us at 1834 MHz  5.8 TB/s                237 us
//   1 token, 777 rows (fp16)           10.5 us
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "paged_common.cuh"
#include "sm100_primitives.cuh"

namespace ngb {
namespace {

constexpr int kTile = 128;         // rows of a query tile
constexpr int kKeys = 64;          // keys of a key tile
constexpr int kAttnThreads = 192;  // 6 warps; two CTAs an SM leave 168 registers a thread
constexpr float kRaise = 8.f;      // growth of the maximum (base 2) that is tolerated
// Probabilities are kept times 2^kLift: fp16 ends at 2^16, which leaves 2^15 for those that
// kRaise lets grow, and at its lower end loses what lies below 2^-25: 2^-32 of the running
// maximum so, and 2^-25 of it without (131,000 keys just below that would be 0.4 % of a row).  bf16
// has the exponents of fp32.
template <bool BF16>
constexpr float kLift = BF16 ? 0.f : 7.f;
constexpr int kItems = 4;          // work items handed out ahead
// Least work of a CTA, in key tiles: few requests are spread wide, but not so that most
// of a CTA's time is its start (one token over 777 rows: 12.0 us with 4, 10.8 with 2, 11.1 with 1;
// over 4000 rows 13.9, 13.4 and 15.4; a tree of 60 over 2000 rows 25.7, 22.4 and 22.4).
constexpr int kMinUnits = 2;
// What an item costs beside its key tiles, in key tiles (32 trees: 110.5 us with 1, 107.3 with 4,
// 106.9 with 6; 1000 short contexts 213, 218 and 221; one token over 100 rows 10.6, 9.1 and 9.1).
constexpr int kItemUnits = 4;

// A work item as one CTA sees it.
struct alignas(16) Item {
  int b, h, i0, ntok;    // request, KV head, tokens [i0, i0 + ntok) of the request
  int first, ctx, kv;    // the request's first token row, rows before its new tokens, all rows
  int need, full;        // keys that the item's tokens need; leading ones that all of them see
  int nt, lo, hi;        // key tiles of the item; this CTA's are [lo, hi); none: the end of the work
  int line;              // of pairs (0), of single tiles (1)
  int pad[3];
};

template <int D>
struct Shape {
  static constexpr int kHalves = D / 64;
  static constexpr int kQBytes = kTile * D * 2, kQHalf = kTile * 128;   // a Q tile, its 64-value half
  static constexpr int kKvBytes = kKeys * D * 2;                        // a K or V tile
  static constexpr int kKvGroup = kHalves * 1024;                       // eight keys of it
  static constexpr int kStages = D == 128 ? 5 : 10;                     // ring: 80 KB
  static constexpr int kSmem = kQBytes + kStages * kKvBytes;
  // One partial: [D / 4][rows, up to a power of two][4] values (a warp, one row a lane, writes
  // 512 bytes in a row), and from the 128 x D-th value on 128 maxima, 128 sums.
  static constexpr size_t kPartFloats = static_cast<size_t>(kTile) * (D + 2);
};

// What the joining kernel needs to know of an item that lies in several CTAs: each of
// them says so for itself, under the slot of its partial (rows 0: none).  Slot 1 holds the
// part of an item that begins in the CTA, slot 0 of one that began before.
struct alignas(16) Meta {
  int rows, token, head;  // token: the first one's row
  int first, parts;       // the CTAs that hold a part: [first, first + parts)
  int pad[3];
};

// How the TMA boxes lie in the cache.  A K or V tile is kept as [group of 8 keys][64-value
// half][8 rows of 128 bytes], so that one box brings whole rows of a page (up to a tile)
// wherever five dimensions can name them: 64 values, 8 rows, halves, groups, and a last
// one that goes through heads and pages alike or has the heads joined to the halves.
// Boxes of 16 rows x 128 bytes, one for each half, were issued too slowly: prompts of
// 16-row pages took 385 us where whole rows took 350, all else alike.  Strides that no such view fits are read in
// boxes of 8 rows and one half (split).
struct BoxPlan {
  int split;
  int head2, page4, head4;  // third coordinate head * head2, fifth page * page4 + head * head4
};

__device__ __forceinline__ int log2_up(int rows) { return 32 - __clz(rows - 1); }

struct TreeAttnArgs {
  const uint16_t* v;
  CacheStrides cs;
  BoxPlan box;
  const int* table;
  long long table_stride;
  int table_width;
  const int* kv_lens;
  const int* cu;
  const unsigned long long* mask;
  int mask_words;
  uint16_t* out;
  float* lse;
  int B, T, Hq, Hkv, G, tok_tile, num_pages, page_shift;
  float scale_log2;
  float* part;
  Meta* meta;
  unsigned int* err;
};

// ---------------------------------------------------------------------------
// The line of work
// ---------------------------------------------------------------------------
struct Request {
  int first, n, kv, ctx;
};

__device__ __forceinline__ Request load_request(const TreeAttnArgs& p, int b) {
  Request r;
  r.first = min(max(p.cu[b], 0), p.T);
  r.n = min(max(p.cu[b + 1], r.first), p.T) - r.first;
  const long long most = static_cast<long long>(p.table_width) << p.page_shift;
  r.kv = max(p.kv_lens[b], 0);
  if (r.kv > most) {  // more rows than its table names
    atomicOr(p.err, kErrBadIndex);
    r.kv = static_cast<int>(most);
  }
  r.ctx = max(0, r.kv - r.n);
  return r;
}

// Keys that the tokens [i0, i1) need, and the leading ones that all of them see.
__device__ __forceinline__ int keys_needed(const TreeAttnArgs& p, const Request& r, int i1) {
  return p.mask ? r.kv : min(r.kv, r.ctx + i1);
}
__device__ __forceinline__ int keys_full(const TreeAttnArgs& p, const Request& r, int i0) {
  return p.mask ? r.ctx : min(r.kv, r.ctx + i0 + 1);
}
__device__ __forceinline__ int tiles_of(int keys) { return max(1, (keys + kKeys - 1) / kKeys); }

// A request's tokens [begin, end) on a line, `stride` for one place of it: whole pairs of
// tiles are on line 0, the last tile of an odd number on line 1.  Without kPairs no
// request has more than one tile, and there is no line 0.
struct Stretch {
  int begin, end, stride;
};
template <bool kPairs>
__device__ __forceinline__ Stretch stretch(const TreeAttnArgs& p, const Request& r, int line) {
  const int step = p.tok_tile;
  if (!kPairs) return Stretch{0, min(r.n, 1) * step, step};
  const int tiles = (r.n + step - 1) / step, paired = (tiles & ~1) * step;
  return line ? Stretch{paired, tiles * step, step} : Stretch{0, paired, 2 * step};
}
// Units of the place at token i0: the key tiles of its last token, and kItemUnits.
__device__ __forceinline__ int place_units(const TreeAttnArgs& p, const Request& r, int i0, int stride) {
  return tiles_of(keys_needed(p, r, min(r.n, i0 + stride))) + kItemUnits;
}
// Units of one KV head of a request.
__device__ __forceinline__ long long head_units(const TreeAttnArgs& p, const Request& r, const Stretch& s) {
  if (s.begin == s.end) return 0;
  if (p.mask || s.end - s.begin == s.stride)
    return static_cast<long long>((s.end - s.begin) / s.stride) * place_units(p, r, s.begin, s.stride);
  long long u = 0;
#pragma unroll 1
  for (int i0 = s.begin; i0 < s.end; i0 += s.stride) u += place_units(p, r, i0, s.stride);
  return u;
}

// a / b for 0 <= a, 0 < b; the 64-bit division is several times as long as the other.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if ((a | b) >> 32) return a / b;
  return static_cast<unsigned>(a) / static_cast<unsigned>(b);
}

// A CTA's way along a line.
template <bool kPairs>
struct Walk {
  long long u, u1;  // next unit, end of the share
  unsigned each;    // units of a share; the first `rest` shares have one more
  int rest, share;  // this CTA's share
  int line;
  int b, h, i0;     // place that u lies in: request, KV head, first token
  int off;          // units of it before u
  int loaded;       // whether r is request b's
  Request r;
  Stretch s;

  // `follow` is where the second line begins.
  __device__ __forceinline__ bool next(const TreeAttnArgs& p, const Walk* follow, Item& it) {
    for (;;) {
      if (u >= u1 || b >= p.B) {
        if (!kPairs || line) return false;
        *this = *follow;
        continue;
      }
      if (!loaded) {
        r = load_request(p, b);
        s = stretch<kPairs>(p, r, line);
        i0 = s.begin;
        loaded = 1;
      }
      if (s.begin == s.end) {
        ++b;
        loaded = 0;
        continue;
      }
      const int t0 = i0 + (!kPairs || line ? 0 : (blockIdx.x & 1) * p.tok_tile);  // the CTAs of a pair take a tile each
      const int i1 = min(r.n, t0 + p.tok_tile);
      const int need = keys_needed(p, r, i1);
      const int units = place_units(p, r, i0, s.stride);
      const int take = static_cast<int>(min(static_cast<long long>(units - off), u1 - u));
      it.b = b, it.h = h, it.i0 = t0, it.ntok = i1 - t0;
      it.first = r.first, it.ctx = r.ctx, it.kv = r.kv, it.need = need, it.full = keys_full(p, r, t0);
      it.nt = tiles_of(need), it.lo = max(0, off - kItemUnits), it.hi = min(it.nt, off + take - kItemUnits);
      it.line = line;
      u += take;
      off += take;
      if (off == units) {
        off = 0;
        i0 += s.stride;
        if (i0 >= s.end) {
          i0 = s.begin;
          if (++h == p.Hkv) {
            h = 0;
            ++b;
            loaded = 0;  // when the next item is asked for: this one should not wait for it
          }
        }
      }
      if (it.hi > it.lo) return true;
    }
  }
};

template <int kStages, bool kPairs>
struct alignas(16) Shared {
  uint64_t full[kStages], empty[kStages];
  uint64_t sfull[2], pfull[2];  // by buffer
  uint64_t qfull, qempty;       // Q is there; the item's last scores are computed
  uint64_t ofull, olast;        // olast: all but the last P V of an item are done
  uint64_t item_full[kItems], item_empty[kItems];
  Item items[kItems];
  long long warp_sum[2][kAttnThreads / 32];
  Walk<kPairs> start[2];        // where this CTA's shares of the lines begin
  uint32_t tmem;
  int abort;
  int bad[2];                   // by parity of the item: its number + 1 if it had V values that are not finite
};

// ---------------------------------------------------------------------------
// PTX used here only
// ---------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const void* tmap, uint64_t* bar, int c0, int c1,
                                            int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* tmap, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}

// One lane of a converged warp.  The MMA warp runs converged, with operands that
// are the same in all lanes, and issues under this predicate: the compiler then
// keeps them in uniform registers, which tcgen05 instructions take.  (Issued from
// a "lane 0" branch instead, every MMA took 140 cycles, twice the tensor core's time.)
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// Shared-memory matrix descriptors, low words (start address >> 4, leading offset
// >> 4 from bit 16) and high words: stride offset (to the next eight 128-byte rows),
// version 1, 128-byte swizzle.
//   K-major (Q, K): rows of 64 values; the leading offset is not used.
//   N-major (V as the B operand, N = the D values contiguous): 8 keys per atom, the
//   stride offset steps along the keys, the leading offset to the next 64 values.
constexpr uint32_t desc_high(int stride) { return (stride >> 4) | (1u << 14) | (2u << 29); }
__device__ __forceinline__ uint32_t desc_kmajor(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_nmajor(uint32_t addr) { return (addr >> 4) | ((1024u >> 4) << 16); }

// Keeps the compiler from computing the operands of all products of an item ahead
// of its loop, which takes more registers than the warp has.
__device__ __forceinline__ void opaque(uint32_t& a, uint32_t& b, uint32_t& c) {
  asm volatile("" : "+r"(a), "+r"(b), "+r"(c));
}

// D[tmem] (+)= A * B, descriptors by their low words; A from shared / from tensor memory.
template <int D>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .b64 x, y;\n\t.reg .pred p;\n\t"
      "mov.b64 x, {%1, %3};\n\tmov.b64 y, {%2, %4};\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "n"(desc_high(1024)), "n"(desc_high(Shape<D>::kKvGroup)), "r"(idesc), "r"(accumulate)
      : "memory");
}
template <int D>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .b64 y;\n\t.reg .pred p;\n\t"
      "mov.b64 y, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "n"(desc_high(Shape<D>::kKvGroup)), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 32 consecutive columns.
__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, float* f) {
  uint32_t* r = reinterpret_cast<uint32_t*>(f);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
      "%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <bool BF16>
__device__ __forceinline__ float value(uint16_t v) {
  return BF16 ? __uint_as_float(static_cast<uint32_t>(v) << 16) : __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Logarithm of a row's sum of exponentials, from its maximum and its sum.
template <bool BF16>
__device__ __forceinline__ float lse_of(float m, float l) {
  constexpr float kUnlift = BF16 ? 1.f : 1.f / 128.f;
  static_assert(kLift<BF16> == (BF16 ? 0.f : 7.f));
  return l == 0.f ? -INFINITY : (m + log2f(l * kUnlift)) * 0.6931471805599453f;
}
__device__ __forceinline__ f2 f2_add(f2 a, f2 b) {
  f2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}

// Bounded wait; false once the CTA has given up.  Plain polling measured fastest: a
// suspend-time hint or a nanosleep between polls adds its wake-up to a chain of short
// hand-overs (one token, 777 rows: 1.5 us more with either).  Kept short, as there are many
// of them, with the low word of the timer (nanoseconds; it wraps after four seconds).  Reading
// it also paces the polls: with the clock instead, the waiting warps took issue slots
// from the others (chains 357 us instead of 343).
__device__ __forceinline__ uint32_t timer_ns() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
  return t;
}
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, unsigned int* err, volatile int* abort) {
  auto poll = [&]() {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
  };
  if (poll()) return true;
  const uint32_t t0 = timer_ns();
  for (;;) {
    if (poll()) return true;
    if (*abort || timer_ns() - t0 > 1000000000u) break;
  }
  atomicOr(err, kErrWaitTimeout);
  *abort = 1;
  return false;
}
// The same for a converged warp.  All lanes poll: one lane's answer would have to be
// passed to the others first.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, unsigned int* err, volatile int* abort) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity, err, abort));
}

// 32 bits of token row `row`'s mask from bit `at` on (which may be negative).
__device__ __forceinline__ uint32_t mask_window(const TreeAttnArgs& p, int row, int at) {
  if (at <= -32) return 0;
  const unsigned long long* m = p.mask + static_cast<size_t>(row) * p.mask_words;
  auto word = [&](int i) { return i < p.mask_words ? m[i] : 0ull; };
  if (at < 0) return static_cast<uint32_t>(word(0) << -at);
  const int w = at >> 6, s = at & 63;
  unsigned long long v = word(w) >> s;
  if (s > 32) v |= word(w + 1) << (64 - s);
  return static_cast<uint32_t>(v);
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// Which of the 32 keys from `key` on token i of the item's request sees.
__device__ __forceinline__ uint32_t visible(const TreeAttnArgs& p, const Item& it, int i, int key) {
  if (!p.mask) return low_bits(min(it.kv, it.ctx + i + 1) - key);
  return (low_bits(it.ctx - key) | mask_window(p, it.first + i, key - it.ctx)) & low_bits(it.kv - key);
}

// ---------------------------------------------------------------------------
// Main kernel
// ---------------------------------------------------------------------------
template <bool BF16, int D, bool kPairs>
__global__ void __launch_bounds__(kAttnThreads, 2)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                     const __grid_constant__ CUtensorMap tmap_tile, const __grid_constant__ CUtensorMap tmap_token,
                     const __grid_constant__ TreeAttnArgs p) {
  using Sh = Shape<D>;
  constexpr int kStages = Sh::kStages, kFirst = kPairs ? 0 : 1;  // kFirst: the first line
  extern __shared__ __align__(1024) unsigned char smem[];  // 1024: the swizzle atom
  unsigned char* ring = smem + Sh::kQBytes;
  auto* sh = reinterpret_cast<Shared<kStages, kPairs>*>(smem + Sh::kSmem);
  volatile int* abort = &sh->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh->sfull[b], 1);
      mbar_init(&sh->pfull[b], 4);
    }
    mbar_init(&sh->qfull, 1);
    mbar_init(&sh->qempty, 1);
    mbar_init(&sh->ofull, 1);
    mbar_init(&sh->olast, 1);
    for (int s = 0; s < kItems; ++s) {
      mbar_init(&sh->item_full[s], 1);
      mbar_init(&sh->item_empty[s], 5);  // MMA, 4 softmax warps
    }
    sh->abort = 0;
    for (int l = 0; l < 2; ++l)  // no work, unless a thread finds some below
      sh->start[l].u = sh->start[l].u1 = 0, sh->start[l].line = l;
    sh->bad[0] = sh->bad[1] = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
    tma_prefetch_desc(&tmap_token);
  }
  if (warp == 5) tmem_alloc(&sh->tmem, 256);
#pragma unroll 1
  for (int c = tid; c < Sh::kQBytes / 16; c += kAttnThreads) reinterpret_cast<uint4*>(smem)[c] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  pdl_launch_next();
  pdl_wait_previous();

  // ---- this CTA's shares of the lines
  const int per = (p.B + kAttnThreads - 1) / kAttnThreads;
  const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
  const int head = min(max(p.cu[0], 0), p.T), tokens = min(max(p.cu[p.B], head), p.T);
  long long mine[2] = {0, 0};
  Request req = {0, 0, 0, 0};
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    req = load_request(p, b);
#pragma unroll
    for (int l = kFirst; l < 2; ++l) mine[l] += head_units(p, req, stretch<kPairs>(p, req, l)) * p.Hkv;
  }
  long long inc[2] = {mine[0], mine[1]};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, inc[0], o), y = __shfl_up_sync(0xffffffffu, inc[1], o);
    if (lane >= o) inc[0] += x, inc[1] += y;
  }
  if (lane == 31) sh->warp_sum[0][warp] = inc[0], sh->warp_sum[1][warp] = inc[1];
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
#pragma unroll 1
  for (int l = kFirst; l < 2; ++l) {
    const long long own = l ? mine[1] : mine[0];
    long long before = (l ? inc[1] : inc[0]) - own, total = 0;
#pragma unroll
    for (int w = 0; w < kAttnThreads / 32; ++w) {
      if (w < warp) before += sh->warp_sum[l][w];
      total += sh->warp_sum[l][w];
    }
    if (total == 0) continue;
    // Shares of at least kMinUnits: some CTAs stay idle when there is little work (the last on
    // the line of pairs, the first on the other).
    const int most = l ? gridDim.x : gridDim.x / 2;
    const int share = l ? gridDim.x - 1 - blockIdx.x : blockIdx.x / 2;
    const int shares = static_cast<int>(min(static_cast<long long>(most), max(1ll, total / kMinUnits)));
    const long long each = quotient(total, shares), rest = total - each * shares;
    const int c = min(share, shares);
    const long long u0 = each * c + min(static_cast<long long>(c), rest);
    const long long u1 = c < shares ? u0 + each + (c < rest) : u0;
    if (u0 < u1 && before <= u0 && u0 < before + own) {
      Walk<kPairs> w;
      w.u = u0, w.u1 = u1, w.loaded = 1, w.line = l, w.share = share;
      w.each = static_cast<unsigned>(min(each, 0xfffffff0ll)), w.rest = static_cast<int>(rest);
      long long o = u0 - before, hu = 0;
#pragma unroll 1
      for (w.b = b0;; ++w.b) {
        if (b1 - b0 > 1) req = load_request(p, w.b);
        w.s = stretch<kPairs>(p, req, l);
        hu = head_units(p, req, w.s);
        if (o < hu * p.Hkv) break;
        o -= hu * p.Hkv;
      }
      w.r = req;
      w.h = static_cast<int>(quotient(o, hu));
      o -= w.h * hu;
#pragma unroll 1
      for (w.i0 = w.s.begin;; w.i0 += w.s.stride) {
        const int units = place_units(p, req, w.i0, w.s.stride);
        if (o < units) break;
        o -= units;
      }
      w.off = static_cast<int>(o);
      sh->start[l] = w;
    }
  }
  __syncthreads();
  // rows in front of the first request's tokens and beyond the last one's see nothing
  const long long row_chunks = static_cast<long long>(p.Hq) * (D / 8), gap = (tokens - head) * row_chunks;
#pragma unroll 1
  for (long long i = static_cast<long long>(blockIdx.x) * kAttnThreads + tid; i < p.T * row_chunks - gap;
       i += static_cast<long long>(gridDim.x) * kAttnThreads) {
    const long long at = i < head * row_chunks ? i : i + gap;
    reinterpret_cast<uint4*>(p.out)[at] = make_uint4(0, 0, 0, 0);
    if (p.lse && at % (D / 8) == 0) p.lse[at / (D / 8)] = -INFINITY;
  }
  const uint32_t tmem = sh->tmem;

  // The item that is k-th in this CTA: waits for it; false when there is none (or
  // the CTA has given up).  done(k) after its last use, one lane of a warp.
  auto item_at = [&](int k) -> const Item& { return sh->items[k % kItems]; };
  auto next_item = [&](int k) {
    return wait_warp(&sh->item_full[k % kItems], (k / kItems) & 1, p.err, abort) && item_at(k).hi > item_at(k).lo;
  };
  auto done = [&](int k) { mbar_arrive(&sh->item_empty[k % kItems]); };

  // Places of the ring in an item of n tiles: K0 K1 V0 K2 V1 K3 ..., the order of the MMAs.
  if (warp == 4) {
    // ------------------------------------------------------------ TMA producer
    const BoxPlan box = p.box;
    const int shift = box.split ? 3 : min(p.page_shift, 6);  // rows of a box: a page, or a whole tile of one
    const int pieces = kKeys >> shift, halves = box.split ? Sh::kHalves : 1;
    const int piece = lane / halves, half = lane % halves;
    const uint32_t piece_bytes = (box.split ? 128u : 2u * D) << shift;
    const uint32_t offset = lane * piece_bytes;
    const int page_mask = (1 << p.page_shift) - 1;
    uint32_t st = 0, ph = 0;  // stage and parity of the next place
    int filled = 0;           // rows of Q in shared memory that may not be zero
    bool ok = true;
    Walk<kPairs> walk = sh->start[kFirst];
    for (int k = 0; ok; ++k) {
      if (!wait_warp(&sh->item_empty[k % kItems], ((k / kItems) & 1) ^ 1, p.err, abort)) break;
      Item it;  // (all lanes walk alike)
      const bool more = walk.next(p, &sh->start[1], it);
      if (!more) it.lo = it.hi = 0;
      if (lane == 0) {
        sh->items[k % kItems] = it;
        mbar_arrive(&sh->item_full[k % kItems]);
      }
      if (!more) break;
      const int n = it.hi - it.lo;
      const int* row = p.table + static_cast<long long>(it.b) * p.table_stride;
      auto key_at = [&](int j) { return (it.lo + j) * kKeys + (piece << shift); };
      auto active_at = [&](int j) { return piece < pieces && j < n && key_at(j) < it.need; };
      auto page_at = [&](int j) { return active_at(j) ? row[key_at(j) >> p.page_shift] : 0; };
      auto load = [&](bool is_v, int j, int page) {
        if (!wait_warp(&sh->empty[st], ph ^ 1, p.err, abort)) return false;
        const bool active = active_at(j);
        const unsigned votes = __ballot_sync(0xffffffffu, active);
        if (lane == 0) mbar_arrive_expect_tx(&sh->full[st], __popc(votes) * piece_bytes);
        __syncwarp();
        if (active) {
          if (page < 0 || page >= p.num_pages) {  // outside the pool: the load fills zeros
            atomicOr(p.err, kErrBadIndex);
            page = p.num_pages;
          }
          const int at = key_at(j) & page_mask;
          tma_load_5d(smem_u32(ring + st * Sh::kKvBytes) + offset, is_v ? &tmap_v : &tmap_k, &sh->full[st], 0,
                      box.split ? at : 0, box.split ? half : it.h * box.head2, box.split ? it.h : at >> 3,
                      page * box.page4 + it.h * box.head4);
        }
        if (++st == kStages) st = 0, ph ^= 1;
        return true;
      };
      // The item's Q rows, a box for a whole tile or one for each token, and zeros in the rows
      // beyond: products with zero take a fraction of the power, and under the power limit
      // of a long decode that is clock rate (64 x 8192 single tokens of 4 rows: 242 -> 224 us).
      // (Loaded by the softmax warps, Q took 2000 to 7000 cycles of an item: 1000 contexts of up
      // to 500 rows 357 us instead of 272.)
      auto load_q = [&]() {
        if (!wait_warp(&sh->qempty, (k & 1) ^ 1, p.err, abort)) return false;
        const int rows = it.ntok * p.G;
#pragma unroll 1
        for (int c = rows * (D / 8) + lane; c < filled * (D / 8); c += 32)
          *reinterpret_cast<uint4*>(smem + (c & 7) * 16 + (c >> 3) % Sh::kHalves * Sh::kQHalf +
                                    (c >> 3) / Sh::kHalves * 128) = make_uint4(0, 0, 0, 0);
        filled = rows;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&sh->qfull, rows * D * 2);
        __syncwarp();
        const bool tile = it.ntok == p.tok_tile;
#pragma unroll 1
        for (int i = lane; i < (tile ? 1 : it.ntok) * Sh::kHalves; i += 32) {
          const int h = i % Sh::kHalves, tk = i / Sh::kHalves;
          tma_load_3d(smem_u32(smem) + h * Sh::kQHalf + tk * p.G * 128, tile ? &tmap_tile : &tmap_token, &sh->qfull,
                      h * 64, it.h * p.G, it.first + it.i0 + tk);
        }
        return true;
      };
      int pg0 = page_at(0), pg1 = page_at(1);  // of tiles j and j + 1
      ok = load(false, 0, pg0) && load_q() && (n == 1 || load(false, 1, pg1));
      for (int j = 0; ok && j < n; ++j) {
        const int pg2 = page_at(j + 2);
        ok = load(true, j, pg0) && (j + 2 >= n || load(false, j + 2, pg2));
        pg0 = pg1;
        pg1 = pg2;
      }
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc_s = umma_idesc_f16(BF16, kTile, kKeys);
    constexpr uint32_t idesc_o = umma_idesc_f16(BF16, kTile, D) | (1u << 16);  // B (V) is N-major
    uint32_t st = 0, ph = 0;      // stage and parity of the next place
    uint32_t q_ph = 0, p_ph = 0;  // parities of Q and of P (bit buffer)
    // broadcasts: known to be the same in all lanes
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t q_desc = __shfl_sync(0xffffffffu, desc_kmajor(smem_u32(smem)), 0);
    const uint32_t ring_k = __shfl_sync(0xffffffffu, desc_kmajor(smem_u32(ring)), 0);
    const uint32_t ring_v = __shfl_sync(0xffffffffu, desc_nmajor(smem_u32(ring)), 0);
    auto advance = [&]() {
      if (++st == kStages) st = 0, ph ^= 1;
    };
    auto scores = [&](int b, bool last) {  // S = Q K^T into buffer b, K at the current place
      if (!wait_warp(&sh->full[st], ph, p.err, abort)) return false;
      tc_fence_after();
      if (elect_one()) {
        uint32_t d = tmem_u + b * kKeys, qd = q_desc, kd = ring_k + st * (Sh::kKvBytes >> 4);
        opaque(d, qd, kd);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          mma_ss<D>(d, qd + (((kk >> 2) * Sh::kQHalf + (kk & 3) * 32) >> 4),
                 kd + (((kk >> 2) * 1024 + (kk & 3) * 32) >> 4), idesc_s, kk != 0);
        umma_commit(&sh->sfull[b]);
        if (last) umma_commit(&sh->qempty);
        umma_commit(&sh->empty[st]);
      }
      __syncwarp();
      advance();
      return true;
    };
    auto values = [&](int b, int j, int n) {  // O += P V, P in buffer b, V at the current place
      if (!wait_warp(&sh->full[st], ph, p.err, abort) || !wait_warp(&sh->pfull[b], (p_ph >> b) & 1, p.err, abort))
        return false;
      p_ph ^= 1u << b;
      tc_fence_after();
      if (elect_one()) {
        uint32_t d = tmem_u + 2 * kKeys, a = tmem_u + b * kKeys, vd = ring_v + st * (Sh::kKvBytes >> 4);
        opaque(d, a, vd);
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          mma_ts<D>(d, a + kk * 8, vd + kk * (2 * Sh::kKvGroup >> 4), idesc_o, kk ? 1u : static_cast<uint32_t>(j != 0));
        umma_commit(&sh->empty[st]);
        if (j == n - 2) umma_commit(&sh->olast);
        if (j == n - 1) umma_commit(&sh->ofull);
      }
      __syncwarp();
      advance();
      return true;
    };
    bool ok = true;
    for (int k = 0; ok && next_item(k); ++k) {
      const Item& it = item_at(k);
      const int n = __shfl_sync(0xffffffffu, it.hi, 0) - __shfl_sync(0xffffffffu, it.lo, 0);
      if (lane == 0) done(k);
      ok = wait_warp(&sh->qfull, q_ph, p.err, abort);
      q_ph ^= 1;
#pragma unroll 1
      for (int t = 0; ok && t < n + 2; ++t) {  // O += P V of tile t - 2, then the scores of tile t
        const int b = t & 1;
        if (t >= 2) ok = values(b, t - 2, n);
        if (ok && t < n) ok = scores(b, t == n - 1);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax, one thread per row
    const int row = tid & (kTile - 1);   // row of the tile
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t ts = tmem + lanes, to = tmem + 2 * kKeys + lanes;  // scores, O
    uint32_t s_ph = 0, o_ph = 0, last_ph = 0;  // parities: S (bit buffer), O, olast
    uint32_t places = 0;                       // ring places of the items before
    bool ok = true;
    const int rt = row / p.G;

    // What no MMA may see of the j-th V tile of an item of n: rows beyond the item's keys
    // become zeros, and so do values that are not finite in rows that some query
    // does not see (true if there are any).  Each softmax warp does 16 rows before it hands on
    // its P, which the product with this tile waits for.  The use of the stage before this one
    // is over: its place lies before that of K_j, whose scores are there; so the
    // parity cannot stand for another use.
    auto clean_values = [&](const Item& x, int k, int n, int j) {
      const uint32_t pl = places + min(n, j + 2) + j, st = pl % kStages;
      ok = wait_warp(&sh->full[st], (pl / kStages) & 1, p.err, abort);
      if (!ok) return;
      unsigned char* tile = ring + st * Sh::kKvBytes;
      bool bad = false;
      const int r = tid >> 1, key = (x.lo + j) * kKeys + r;  // two threads a row
      if (key >= x.full) {
        const bool beyond = key >= x.need;
#pragma unroll 2
        for (int q = 0; q < D / 16; ++q) {
          const int c = q * 2 + (tid & 1);  // 16-byte chunk of the row
          uint4* at = reinterpret_cast<uint4*>(tile + (r >> 3) * Sh::kKvGroup + (c >> 3) * 1024 + (r & 7) * 128 + (((c + r) & 7) << 4));
          if (beyond) {
            *at = make_uint4(0, 0, 0, 0);
            continue;
          }
          const uint4 v = *at;
          constexpr uint32_t kExp = BF16 ? 0x7F807F80u : 0x7C007C00u, kOne = BF16 ? 0x00800080u : 0x04000400u;
          auto infinite = [&](uint32_t u) { return ((u & kExp) + kOne) & 0x80008000u; };
          if (infinite(v.x) | infinite(v.y) | infinite(v.z) | infinite(v.w)) {
            auto clear = [&](uint32_t u) {
              const uint32_t f = infinite(u);
              return u & ~((f & 0x8000u ? 0xFFFFu : 0u) | (f & 0x80000000u ? 0xFFFF0000u : 0u));
            };
            *at = make_uint4(clear(v.x), clear(v.y), clear(v.z), clear(v.w));
            bad = true;
          }
        }
      }
      if (bad) sh->bad[k & 1] = k + 1;
      fence_proxy_async_smem();
    };

    bool more = next_item(0);
    // Where the partials and their descriptions lie: the shares of the even tiles, of the
    // odd ones, of the line of single tiles.
    const int place0 = (blockIdx.x & 1) * (gridDim.x / 2) + blockIdx.x / 2, place1 = 2 * gridDim.x - 1 - blockIdx.x;
    if (tid < 4) p.meta[2 * (tid & 2 ? place1 : place0) + (tid & 1)] = Meta{};
    __syncwarp();
    for (int k = 0; more; ++k) {
      const Item& it = item_at(k);
      const int n = it.hi - it.lo, lo = it.lo, full = it.full;
      const int rows = it.ntok * p.G;
      const bool busy = warp * 32 < rows;  // this warp has rows
      const bool live = row < rows;
      const int my_token = it.i0 + (live ? rt : 0);
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j) {
        const int b = j & 1;
        ok = wait_warp(&sh->sfull[b], (s_ph >> b) & 1, p.err, abort);
        if (!ok) break;
        s_ph ^= 1u << b;
        tc_fence_after();
        if (busy) {
          const int key0 = (lo + j) * kKeys;
          const f2 scale2 = f2_make(p.scale_log2, p.scale_log2);
          float x[kKeys];
          uint32_t w[kKeys / 2];
          f2 sum;
          tmem_ld_32(ts + b * kKeys, x);
          tmem_ld_32(ts + b * kKeys + 32, x + 32);
          tmem_ld_wait();
          if (key0 + kKeys > full) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t vis = live ? visible(p, it, my_token, key0 + 32 * h) : 0u;
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (!((vis >> c) & 1)) x[32 * h + c] = -INFINITY;
            }
          }
          float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int c = 4; c < kKeys; c += 8) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mx[q] = c + 4 + q < kKeys ? fmaxf(fmaxf(mx[q], x[c + q]), x[c + 4 + q]) : fmaxf(mx[q], x[c + q]);
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
          if (j == 0) {
            m = top;
          } else if (const bool raise = live && top > m + kRaise; __any_sync(0xffffffffu, raise)) {
            // O must hold all tiles before this one: the next scores were issued after P V
            // of the tile before; at the last tile olast says so.
            ok = j + 1 < n ? wait_warp(&sh->sfull[b ^ 1], (s_ph >> (b ^ 1)) & 1, p.err, abort)
                            : wait_warp(&sh->olast, last_ph, p.err, abort);
            if (!ok) break;
            tc_fence_after();
            // each row by its own values alone, whatever the rows beside it do
            const float f = !raise ? 1.f : m == -INFINITY ? 0.f : exp2_approx(m - top);
            m = raise ? top : m;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_ld_16(to + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int q = 0; q < 16; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * f);
              tmem_st_16(to + c, o);
            }
          }
          const float base = !live ? -INFINITY : m == -INFINITY ? 0.f : kLift<BF16> - m;  // (no row: P = 0)
          const f2 base2 = f2_make(base, base);
          f2 sums[2] = {f2_make(0.f, 0.f), f2_make(0.f, 0.f)};
#pragma unroll
          for (int q = 0; q < kKeys / 2; ++q) {
            float a, c;
            f2_split(f2_fma(f2_make(x[2 * q], x[2 * q + 1]), scale2, base2), a, c);
            a = exp2_approx(a);
            c = exp2_approx(c);
            sums[q & 1] = f2_add(sums[q & 1], f2_make(a, c));
            w[q] = pack_pair<BF16>(a, c);
          }
          tmem_st_16(ts + b * kKeys, w);
          tmem_st_16(ts + b * kKeys + 16, w + 16);
          sum = f2_add(sums[0], sums[1]);
          float a, c;
          f2_split(sum, a, c);
          l += a + c;
          tmem_st_wait();
        }
        if ((lo + j + 1) * kKeys > full) {
          clean_values(it, k, n, j);
          if (!ok) break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->pfull[b]);
      }
      if (!ok) break;
      places += 2 * n;
      more = next_item(k + 1);

      // ---- the item's end
      const bool whole = lo == 0 && it.hi == it.nt;
      const int slot = lo > 0 ? 0 : 1;
      const int place = !kPairs || it.line ? place1 : place0;
      if (!whole && tid == 0) {  // the shares that hold the tiles before and after this one's
        const Walk<kPairs>& from = sh->start[kPairs ? it.line : 1];
        const unsigned each = from.each;
        const int c = from.share, rest = from.rest;  // shares before `rest` have one unit more
        auto shares = [&](unsigned tiles, int near, unsigned size, unsigned far) {  // `near` of one size, then others
          const unsigned long long most = static_cast<unsigned long long>(near) * size;
          return static_cast<int>(tiles <= most ? (tiles + size - 1) / size
                                                : near + (tiles - static_cast<unsigned>(most) + far - 1) / far);
        };
        const int back = shares(lo, max(0, c - rest), each, each + 1);
        const int ahead = shares(it.nt - it.hi, max(0, rest - c - 1), each + 1, each);
        p.meta[2 * place + slot] = Meta{rows, it.first + it.i0, it.h, place - back, back + ahead + 1, {}};
      }
      ok = wait_warp(&sh->ofull, o_ph, p.err, abort);
      if (!ok) break;
      o_ph ^= 1;
      if (n > 1) last_ph ^= 1;  // (completed before ofull)
      tc_fence_after();
      if (busy) {
        const float norm = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        const size_t out_row = static_cast<size_t>(it.first + my_token) * p.Hq + it.h * p.G + (row - rt * p.G);
        float* part = p.part + (static_cast<size_t>(place) * 2 + slot) * Sh::kPartFloats;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tmem_ld_32(to + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 32; ++q) o[q] *= norm;
          if (!live) continue;
          if (whole) {
            uint4* dst = reinterpret_cast<uint4*>(p.out + out_row * D + c);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              dst[q] = make_uint4(pack_pair<BF16>(o[8 * q], o[8 * q + 1]), pack_pair<BF16>(o[8 * q + 2], o[8 * q + 3]),
                                  pack_pair<BF16>(o[8 * q + 4], o[8 * q + 5]),
                                  pack_pair<BF16>(o[8 * q + 6], o[8 * q + 7]));
          } else {
            const int lg = log2_up(rows);
            float4* dst = reinterpret_cast<float4*>(part) + ((c / 4) << lg) + row;
#pragma unroll
            for (int q = 0; q < 8; ++q) dst[q << lg] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
          }
        }
        // Values that were kept out of the MMA: infinities and NaNs, so they may as well be
        // added to what has been written.
        if (sh->bad[k & 1] == k + 1 && live) {
#pragma unroll 1
          for (int key = max(full, lo * kKeys); key < min(it.need, it.hi * kKeys); ++key) {
            const int page = p.table[static_cast<long long>(it.b) * p.table_stride + (key >> p.page_shift)];
            if (page < 0 || page >= p.num_pages || !(visible(p, it, my_token, key) & 1)) continue;
            const uint16_t* v = p.v + page * p.cs.page + (key & ((1 << p.page_shift) - 1)) * p.cs.row + it.h * p.cs.head;
#pragma unroll 1
            for (int c = 0; c < D; ++c) {
              const float e = value<BF16>(v[c]);
              if (isfinite(e)) continue;
              uint16_t* o16 = p.out + out_row * D + c;
              float* o32 = part + (((c >> 2) << log2_up(rows)) + row) * 4 + (c & 3);
              if (whole)
                *o16 = static_cast<uint16_t>(pack_pair<BF16>(value<BF16>(*o16) + e, 0.f));
              else
                *o32 += e;
            }
          }
        }
        if (live) {
          if (!whole) {
            part[kTile * D + row] = m;
            part[kTile * D + kTile + row] = l;
          } else if (p.lse) {
            p.lse[out_row] = lse_of<BF16>(m, l);
          }
        }
      }
      tc_fence_before();  // O has been read: the next P may be handed on
      __syncwarp();
      if (lane == 0) done(k);
    }
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (*abort) {  // let the TMA copies still in flight land (they take microseconds)
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) {
    }
  }
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// Joins the partials of the items that lie in several CTAs, in a fixed order.  One thread
// has 8 values of a row, rows fastest, as the partials lie.  Block (c, y) works for one of
// the two items that CTA c may hold a part of (y & 1): an item's elements are divided
// evenly among the blocks of its CTAs, so that a few items of many parts keep all SMs busy and
// no block is launched for nothing.  Many parts are shared by the warps of a block.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kJoinFew = 2;

// A softmax-weighted sum of 8 values: maximum, sum, values.
struct Joined {
  float m, l, v[8];
  __device__ __forceinline__ void add(float m2, float l2, const float* v2) {
    if (m2 == -INFINITY) return;
    const float top = fmaxf(m, m2), f = exp2_approx(m - top), f2 = exp2_approx(m2 - top);
    m = top;
    l = l * f + l2 * f2;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * f + v2[i] * f2;
  }
};

template <bool BF16, int D, bool kPairs>
__global__ void __launch_bounds__(kJoinThreads) tree_attn_join(const TreeAttnArgs p) {
  __shared__ float box[kJoinWarps][10][32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_next();
  pdl_wait_previous();
  const Meta single = p.meta[2 * (blockIdx.x + gridDim.x) + (blockIdx.y & 1)];
  Meta mt = kPairs ? p.meta[2 * blockIdx.x + (blockIdx.y & 1)] : single;
  bool filled = false;  // the box is in use
#pragma unroll 1
  for (int line = kPairs ? 0 : 1; line < 2; ++line, mt = single) {
    if (mt.rows == 0) continue;
    const bool many = mt.parts > kJoinFew;
    const int lg = log2_up(mt.rows);
    const int k0 = many ? warp : 0, step = many ? kJoinWarps : 1, pass = many ? 32 : kJoinThreads;
    const int all = (D / 8) << lg, own = ((all + mt.parts - 1) / mt.parts + 31) & ~31;
    const int begin = (static_cast<int>(blockIdx.x + line * gridDim.x) - mt.first) * own, end = min(all, begin + own);
    for (int e0 = begin + (blockIdx.y >> 1) * pass; e0 < end; e0 += (gridDim.y >> 1) * pass) {
      const int e = e0 + (many ? lane : tid), row = e & ((1 << lg) - 1), chunk = e >> lg;
      const bool mine = row < mt.rows && e < end;
      Joined j{-INFINITY, 0.f, {}};
      if (mine) {
#pragma unroll 1  // (four at a time: more code to fetch, 0.3 us on a small call, and no less for 37 parts)
        for (int k = k0; k < mt.parts; k += step) {
          const float* src = p.part + (static_cast<size_t>(mt.first + k) * 2 + (k == 0)) * Shape<D>::kPartFloats;
          const float4* v = reinterpret_cast<const float4*>(src) + (chunk << (lg + 1)) + row;
          const float4 a = v[0], b = v[1 << lg];
          const float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
          j.add(src[kTile * D + row], src[kTile * D + kTile + row], w);
        }
      }
      if (many) {
        if (filled) __syncthreads();
        filled = true;
        box[warp][0][lane] = j.m;
        box[warp][1][lane] = j.l;
#pragma unroll
        for (int i = 0; i < 8; ++i) box[warp][2 + i][lane] = j.v[i];
        __syncthreads();
        if (warp) continue;
        for (int w = 1; w < kJoinWarps; ++w) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = box[w][2 + i][lane];
          j.add(box[w][0][lane], box[w][1][lane], v);
        }
      }
      if (!mine) continue;
      const float inv = j.l == 0.f ? 0.f : 1.f / j.l;
      const int tk = row / p.G;
      const size_t r = static_cast<size_t>(mt.token + tk) * p.Hq + mt.head * p.G + (row - tk * p.G);
      *reinterpret_cast<uint4*>(p.out + r * D + chunk * 8) =
          make_uint4(pack_pair<BF16>(j.v[0] * inv, j.v[1] * inv), pack_pair<BF16>(j.v[2] * inv, j.v[3] * inv),
                     pack_pair<BF16>(j.v[4] * inv, j.v[5] * inv), pack_pair<BF16>(j.v[6] * inv, j.v[7] * inv));
      if (p.lse && chunk == 0) p.lse[r] = lse_of<BF16>(j.m, j.l);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
BoxPlan plan_boxes(const CacheStrides& cs, int D, int Hkv, int pages) {
  if (D == 64) return {0, 1, 1, 0};
  if (cs.head == D || Hkv == 1) return {0, 2, 1, 0};         // a row of all heads is one run of halves
  if (cs.page == cs.head * Hkv && static_cast<long long>(pages) * Hkv < (1LL << 31))
    return {0, 0, Hkv, 1};                                   // heads go on from page to page
  return {1, 0, 1, 0};
}

int make_cache_map(const void* base, const CacheStrides& cs, const BoxPlan& plan, int D, int rows, int Hkv, int pages,
                   CUtensorMap* m) {
  auto enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encode_fn());
  if (!enc) return NG_ERR_CUDA;
  const cuuint64_t u = 2, heads = Hkv, groups = rows / 8;
  const cuuint64_t row = cs.row * u, head = cs.head * u, page = cs.page * u;
  const cuuint32_t halves = D / 64, most = std::min(rows, kKeys) / 8;
  cuuint64_t dims[5] = {64, 8, halves, groups, static_cast<cuuint64_t>(pages)};
  cuuint64_t strides[4] = {row, 128, 8 * row, page};
  cuuint32_t box[5] = {64, 8, halves, most, 1};
  const cuuint32_t es[5] = {1, 1, 1, 1, 1};
  if (plan.split) {
    dims[1] = rows, dims[3] = heads, strides[2] = head;
    box[2] = box[3] = 1;
  } else if (plan.head4) {
    dims[4] *= heads, strides[3] = head;
  } else {
    dims[2] *= heads;
    if (halves == 1) strides[1] = head;
  }
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, const_cast<void*>(base), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? NG_OK
             : NG_ERR_CUDA;
}

// Q, in boxes of `tokens` tokens of one KV head's query heads.
int make_q_map(const void* base, long long token, long long head, int D, int Hq, int T, int G, int tokens, CUtensorMap* m) {
  auto enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encode_fn());
  if (!enc) return NG_ERR_CUDA;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(Hq), static_cast<cuuint64_t>(T)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(Hq > 1 ? head : D) * 2, static_cast<cuuint64_t>(T > 1 ? token : D) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(tokens)};
  const cuuint32_t es[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? NG_OK
             : NG_ERR_CUDA;
}

constexpr size_t kMetaBytes = 65536;
size_t attn_workspace_bytes(int D, const DeviceInfo& dev) {
  const size_t part = D == 128 ? Shape<128>::kPartFloats : Shape<64>::kPartFloats;
  return kMetaBytes + static_cast<size_t>(dev.sm_count) * 8 * part * sizeof(float);  // CTAs x lines x slots
}

template <bool BF16, int D, bool kPairs>
int launch_tree_attn(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mtile, const CUtensorMap& mtoken,
                     const TreeAttnArgs& a, const DeviceInfo& dev,
                     cudaStream_t st) {
  constexpr int smem = Shape<D>::kSmem + static_cast<int>(sizeof(Shared<Shape<D>::kStages, kPairs>));
  static_assert(2 * (smem + 1024) <= 228 * 1024, "two CTAs must fit in the shared memory of an SM");
  const int ctas = 2 * dev.sm_count;
  auto kern = tree_attn_kernel<BF16, D, kPairs>;
  static std::once_flag once[kMaxDevices];
  std::call_once(once[dev.device],
                 [&] { cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (int e = launch_chained(kern, dim3(ctas), dim3(kAttnThreads), smem, st, mk, mv, mtile, mtoken, a)) return e;
  // The shares of an item of 128 rows in two parts are 1024 elements; two passes each.
  const int rows = static_cast<int>(std::min<long long>(kTile, static_cast<long long>(a.T) * a.G));
  return launch_chained(tree_attn_join<BF16, D, kPairs>, dim3(ctas, 2 * ((rows * (D / 8) + 1023) / 1024)), dim3(kJoinThreads), 0, st,
                        a);
}

}  // namespace
}  // namespace ngb

extern "C" size_t ng_tree_attn_workspace_bytes(int D) {
  using namespace ngb;
  DeviceInfo dev;
  if ((D != 64 && D != 128) || current_device_info(&dev) != NG_OK) return 0;
  return attn_workspace_bytes(D, dev);
}

extern "C" int ng_tree_attn(const void* q, long long q_stride_token, long long q_stride_head,
                            const void* k_cache, const void* v_cache, long long stride_page,
                            long long stride_row, long long stride_head, const int* block_table,
                            long long table_stride, int table_width, const int* kv_lens, const int* cu_new,
                            const long long* mask, int mask_words, void* out, float* lse, int dtype, int B,
                            int T, int Hq, int Hkv, int D, int num_pages, int page_size, float scale,
                            void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ngb;
  if (!q || !k_cache || !v_cache || !block_table || !kv_lens || !cu_new || !out || !workspace)
    return NG_ERR_NULL_POINTER;
  if (!act_dtype_ok(dtype)) return NG_ERR_BAD_DTYPE;
  if (B < 1 || T < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || Hq / Hkv > kTile || (D != 64 && D != 128) ||
      num_pages < 1 || table_width < 1 || table_stride < table_width || !page_size_ok(page_size) ||
      static_cast<long long>(T) * Hq > (1LL << 30))
    return NG_ERR_BAD_SHAPE;
  const CacheStrides cs{stride_page, stride_row, stride_head};
  if (!cache_strides_ok(cs) || q_stride_token % 8 || q_stride_head % 8 || q_stride_token < 0 || q_stride_head < 0)
    return NG_ERR_BAD_SHAPE;
  if (!(scale > 0.f) || !(scale < INFINITY) || mask_words < 0 || (mask && mask_words < 1))
    return NG_ERR_BAD_ARGUMENT;
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(out, 16) ||
      !aligned(mask, 8) || !aligned(workspace, 256))
    return NG_ERR_MISALIGNED;
  DeviceInfo dev;
  if (int st = current_device_info(&dev)) return st;
  if (workspace_bytes < attn_workspace_bytes(D, dev)) return NG_ERR_BAD_ARGUMENT;
  CUtensorMap mk, mv, mtile, mtoken;
  const BoxPlan box = plan_boxes(cs, D, Hkv, num_pages);
  if (int st = make_cache_map(k_cache, cs, box, D, page_size, Hkv, num_pages, &mk)) return st;
  if (int st = make_cache_map(v_cache, cs, box, D, page_size, Hkv, num_pages, &mv)) return st;
  const int G = Hq / Hkv;
  if (int st = make_q_map(q, q_stride_token, q_stride_head, D, Hq, T, G, kTile / G, &mtile)) return st;
  if (int st = make_q_map(q, q_stride_token, q_stride_head, D, Hq, T, G, 1, &mtoken)) return st;
  const TreeAttnArgs a{static_cast<const uint16_t*>(v_cache), cs, box, block_table, table_stride, table_width, kv_lens,
                       cu_new, reinterpret_cast<const unsigned long long*>(mask), mask_words,
                       static_cast<uint16_t*>(out), lse, B, T, Hq, Hkv, G, kTile / G, num_pages,
                       log2_of(page_size), scale * 1.4426950408889634f,
                       reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + kMetaBytes),
                       static_cast<Meta*>(workspace), dev.err};
  auto st = static_cast<cudaStream_t>(stream);
  // As many tokens as one tile holds: no request has two tiles, and the kernel without the
  // line of pairs starts sooner (one token, 777 rows: 10.8 us instead of 11.6).
  auto launch = [&](auto bf16, auto dim) {
    return T <= a.tok_tile ? launch_tree_attn<bf16.value, dim.value, false>(mk, mv, mtile, mtoken, a, dev, st)
                           : launch_tree_attn<bf16.value, dim.value, true>(mk, mv, mtile, mtoken, a, dev, st);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (D == 128) return dtype == NG_DTYPE_BF16 ? launch(std::true_type{}, D128{}) : launch(std::false_type{}, D128{});
  return dtype == NG_DTYPE_BF16 ? launch(std::true_type{}, D64{}) : launch(std::false_type{}, D64{});
}
