// Decode attention over the 8-bit paged cache.
//
// Per (slot, KV head, pass of up to 8 kNT query heads) - a segment - with scores in
// base 2: s_t = sm_scale log2(e) key_scale (q . code_t), and a reference m,
//   l <- l + sum_t 2^(s_t - m),   O <- O + value_scale sum_t 2^(s_t - m) code_t.
// The reference is a maximum seen so far, and stays while no score is more than kSlack
// above it: then the weights need no maximum over the warp and O and l no rescaling, which
// were a sixth of the instructions and the longest chain of a tile.
//
// What bounds it: every cached byte is used by g = Hq / H query heads, 4 g flops a byte
// (g = 4 ... 16), so it is a read of the cache at HBM speed.  The arithmetic runs on
// mma.sync m16n8k16 with tokens (scores) or channels (output) as the 16 rows and the
// query heads as the 8 columns: a warp's share of the SM's bandwidth needs a few
// percent of the tensor rate, and the operands can then go from global memory to
// registers without a stop in shared memory:
//   - scores contract over channels, whose order is free as long as q has the same: a
//     lane loads 16 consecutive bytes of its token's row and feeds them, four channels a
//     k-step, to the k indices that the fragment gives it;
//   - outputs contract over tokens: a lane loads 16 consecutive channels of its four
//     tokens of a k-step and pairs the tokens' bytes with byte permutes; the rows of the
//     16 x 8 tile are those channels in an order that only the store undoes;
//   - the weights go from the score tile's layout (token rows, head columns) to the
//     other operand's by a transposing matrix move inside the warp.
// 8-bit codes become fp16 exactly (e4m3 by conversion, int8 by the exponent trick), so
// the products are exact and the sums float32.  q is fp16; a bf16 q is scaled by a power
// of two per head that puts its largest element near the top of fp16's range, which
// keeps elements down to 2^-29 of it exact.  A weight is the sum of fp16 parts, two of 11 bits:
// off by at most 2^-22 of itself or 2^-31 of the one at the reference (bf16 tails: three
// parts of 8 bits).  With one part, 2^-12, the bf16 outputs over 32 x 32K tokens are 6e-4
// (root mean square) from those of float32 weights, so 6e-5.  The second part costs 1 % there in
// a burst (329 us against 326) and 8 % at the clocks of the power cap (380 against 352), with 16
// query heads on a KV head 18 % (462 against 390).
//
// All segments' tiles (kTile tokens of a page, half as many of a tail: about the same
// bytes) are laid end to end, each segment's behind kSetup units that stand for what a
// segment costs a warp besides its tiles, and every warp of a fixed grid takes one
// contiguous slice of the units; warps never wait for one another over the data.  The
// next tile's keys are requested when this tile's scores are done, its values when this
// tile's output is.  A segment inside one slice is stored at once; of one that crosses
// slices every warp leaves a part in the workspace (two places a warp), or, where all
// warps of a CTA work on it, the CTA leaves one, and merge_kernel joins them.
#include "kv8_common.cuh"

namespace kitty8 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHead = 6.f;           // weights are 2^(score - m + kHead): at most 2^(kHead + kSlack) = 2^14, and
constexpr float kSlack = 8.f;          // normal in fp16 down to 2^-20 of the one at m
constexpr float kFar = 1048576.f;      // references beyond this: a product is rounded before the reference is taken off
constexpr float kUnset = -3.402823466e38f;   // no reference yet: any finite score is far above it
constexpr int kWarps = 4;              // per CTA
constexpr int kSetup = 2;              // units (tiles) that beginning and ending a segment count as
constexpr int kAhead = 4;              // tiles that a prefetch asks for
constexpr int kMergeThreads = 256;

// What attention_kernel leaves about a segment for merge_kernel.
struct alignas(16) Note {
  int64_t begin;                       // its first unit, where it left parts
  int64_t units;                       // its units; 0: an empty slot; -1: stored already
};

struct Plan {
  int passes, pass_heads;              // query heads of a KV head in passes of pass_heads
  uint32_t per_page;                   // 2^31 / (page_size / 32), rounded up: see blocks_of
  int warps;                           // of the whole grid
  float* part_ml;                      // [2 warps][pass_heads][2]  reference, sum
  float* part_o;                       // [2 warps][pass_heads][D]
  Note* notes;                         // [segments + 1], the last holding the units of a slice
};

// Read once, past L1.  (Not as read-only data: this kernel may have been launched before the
// one that writes it was done.)
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream2(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <bool kBf16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The four codes of a word as two fp16 pairs.  int8: 0x6400 | (x + 128) is the fp16
// number 1024 + 128 + x, exact, and 1152 is taken off.
template <int kCode>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kCode == KITTY_KV8_E4M3) {
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    const uint32_t x = w ^ 0x80808080u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(prmt(x, 0x64646464u, 0x4140)), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(prmt(x, 0x64646464u, 0x4342)), "r"(0x64806480u));
  }
}

// Tokens of a tile of a page.
template <int kDim>
constexpr int kTileOf = kDim == 256 ? 16 : 32;

// Tiles of a slot's segments: its whole pages, then its tail.
struct Tiles {
  int paged, all, tail;                // tiles in pages, all tiles, tail tokens
  __device__ int units() const { return all ? all + kSetup : 0; }
};
// Whole pages of len >= 0 tokens: (len / 32) / k for pages of 32 k tokens, k <= 8, by a
// product.  With c = ceil(2^31 / k) = (2^31 + e) / k, e < k, and n = len / 32 < 2^26,
// n c / 2^31 is above n / k by n e / (k 2^31) < 1 / k, so it has the same whole part.
__device__ __forceinline__ int blocks_of(const Plan& plan, int len) {
  return int(__umulhi(uint32_t(len) >> 5 << 1, plan.per_page));
}
template <int kTile>
__device__ __forceinline__ Tiles tiles_of(const KittyKv8Cache& c, const Plan& plan, int len) {
  const int blocks = blocks_of(plan, len), tail = len - blocks * c.page_size;
  const int paged = blocks * (c.page_size / kTile);
  return Tiles{paged, paged + (tail + kTile / 2 - 1) / (kTile / 2), tail};
}
// Tokens of batch row b: 0 for padding (a negative slot), and where its slot or its length is
// out of range.  kL2: from L2, for merge_kernel, which asks before it has waited; the SM's L1 may
// hold what was there before the last kernel on the stream.
template <bool kL2 = false>
__device__ __forceinline__ int tokens_of(const KittyKv8AttentionArgs& a, const Plan& plan, int b, uint32_t* err = nullptr) {
  const auto get = [](const int32_t* p) { return kL2 ? __ldcg(p) : *p; };
  const int s = a.seq_map ? get(a.seq_map + b) : b;
  if (s < 0) return 0;
  if (s >= a.cache.slots) {
    if (err) dev::flag(err, kErrSlot);
    return 0;
  }
  const int len = get(a.cache.lengths + s);
  if (len >= 0 && blocks_of(plan, len) <= a.cache.max_pages) return len;
  if (err) dev::flag(err, kErrLength);
  return 0;
}

// a / b for non-negative a and positive b, in 32 bits where they fit (the 64-bit quotient is
// a long sequence on the way to a warp's first load).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}

// Row b has `per_row` = H * passes segments of equal length.
template <int kTile, bool kL2 = false>
__device__ __forceinline__ int units_of_row(const KittyKv8AttentionArgs& a, const Plan& plan, int b,
                                            uint32_t* err = nullptr) {
  return b < a.batch ? tiles_of<kTile>(a.cache, plan, tokens_of<kL2>(a, plan, b, err)).units() : 0;
}

// The rows before a place, in units: thread t of a CTA has rows [t rows_each, (t + 1)
// rows_each).  For batches of more than kFew rows.
struct Rows {
  int64_t before[kWarps * 32];         // units of the rows before each thread's
  int64_t total[kWarps];
};

// By the whole CTA: fills `s`; returns the units of all rows.  The first CTA also flags rows
// whose slot or length is out of range, and notes empty ones.
template <int kTile>
__device__ __forceinline__ int64_t scan_rows(const KittyKv8AttentionArgs& a, const Plan& plan, int per_row,
                                             int rows_each, Rows& s, uint32_t* err) {
  const int tid = threadIdx.x, lane = tid & 31;
  int64_t mine = 0;
#pragma unroll 4
  for (int i = 0; i < rows_each; ++i) {
    const int b = tid * rows_each + i, n = units_of_row<kTile>(a, plan, b, blockIdx.x == 0 ? err : nullptr);
    mine += n;
    if (blockIdx.x == 0 && n == 0 && b < a.batch)
      for (int k = 0; k < per_row; ++k) plan.notes[int64_t(b) * per_row + k].units = 0;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s.total[tid >> 5] = incl;
  __syncthreads();
  int64_t before = incl - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < tid >> 5) before += s.total[w];
    all += s.total[w];
  }
  s.before[tid] = before;
  __syncthreads();
  return all;
}

struct Place {
  int64_t begin;       // first unit of the segment found
  int b, seg;          // its batch row and its index among the row's segments
};
// The same for at most kFew rows, by every warp for itself: no barrier and no second look at the
// lengths.  Lane t has row t.  8 sequences of up to 60 tokens take 8.7 us so and 8.9 by the whole
// CTA, 32 take 9.5 and 9.7; with several rows a lane it is the slower one (64 sequences 11.6 and
// 11.3, 256 of up to 8192 tokens 57.2 and 56.7).
constexpr int kFew = 32;
struct FewRows {
  int one;                             // units of each segment of the row
  int64_t before;                      // units of one segment of each of the rows before it
};
// Returns the units of all rows (one segment of each).
template <int kTile>
__device__ __forceinline__ int64_t scan_few(const KittyKv8AttentionArgs& a, const Plan& plan, int per_row, FewRows& r,
                                            uint32_t* err) {
  const int b = threadIdx.x & 31;
  r.one = units_of_row<kTile>(a, plan, b, blockIdx.x == 0 && threadIdx.x < 32 ? err : nullptr);
  if (blockIdx.x == 0 && threadIdx.x < 32 && r.one == 0 && b < a.batch)
    for (int k = 0; k < per_row; ++k) plan.notes[int64_t(b) * per_row + k].units = 0;
  int64_t incl = r.one;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (b >= o) incl += v;
  }
  r.before = incl - r.one;
  return __shfl_sync(0xffffffffu, incl, 31);
}
__device__ __forceinline__ Place locate_few(int per_row, const FewRows& r, int64_t f) {
  int64_t at = r.before * per_row;
  const uint32_t hit = __ballot_sync(0xffffffffu, f >= at && f < at + int64_t(r.one) * per_row);
  const int src = __ffs(hit) - 1, len = __shfl_sync(0xffffffffu, r.one, src);
  at = __shfl_sync(0xffffffffu, at, src);
  const int seg = int(quotient(f - at, len));
  return Place{at + int64_t(seg) * len, src, seg};
}

// By the whole warp: the segment that holds unit f (less than there are).
template <int kTile>
__device__ __forceinline__ Place locate(const KittyKv8AttentionArgs& a, const Plan& plan, int per_row, int rows_each,
                                        const Rows& s, int64_t f) {
  const int lane = threadIdx.x & 31;
  int found = 0;                       // threads whose rows begin at or before f
#pragma unroll
  for (int w = 0; w < kWarps; ++w) found += __popc(__ballot_sync(0xffffffffu, s.before[w * 32 + lane] * per_row <= f));
  const int b0 = (found - 1) * rows_each;
  Place r{0, b0, 0};
  int64_t before = s.before[found - 1] * per_row;
  for (int i = 0; i < rows_each; i += 32) {
    const int one = i + lane < rows_each ? units_of_row<kTile>(a, plan, b0 + i + lane) : 0;
    int64_t incl = int64_t(one) * per_row;
    const int64_t mine = incl;
    if (rows_each > 1) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
    }
    const int64_t start = before + incl - mine;
    const uint32_t hit = __ballot_sync(0xffffffffu, f >= start && f < start + mine);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int64_t at = __shfl_sync(0xffffffffu, start, src);
      const int len = __shfl_sync(0xffffffffu, one, src);
      r.b = b0 + i + src;
      r.seg = int(quotient(f - at, len));
      r.begin = at + int64_t(r.seg) * len;
      return r;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return r;
}

// Whether all warps of a CTA work on tiles of the segment [begin, end) only.
__device__ __forceinline__ bool cta_inside(int64_t cta, int64_t per_warp, int64_t begin, int64_t end) {
  return cta * kWarps * per_warp >= begin + kSetup && (cta + 1) * kWarps * per_warp <= end;
}

// Warps hide one another's latency, so the registers are capped for 12 warps an SM at 128
// channels (32 x 32K tokens take 325 us, 341 with 8 warps and 432 with 16, 16 x 131K 664, 750 and
// 826) and 16 at 64 (256 mixed lengths 57 us, 62 with 12 warps and 65 with 20).  Under the
// cap 80 to 104 bytes a thread are spilled at 128 channels.
template <int kDim>
constexpr int kMinCtas = kDim == 64 ? 4 : kDim == 128 ? 3 : 1;

// kDim: 64, 128 or 256 channels in registers; kWhole: head_dim == kDim (else the missing
// channels read as zero).  kNT: tiles of 8 query heads.
template <int kDim, int kNT, bool kWhole, bool kBf16, int kCode>
__global__ void __launch_bounds__(kWarps * 32, kNT == 1 ? kMinCtas<kDim> : 1)
    attention_kernel(KittyKv8AttentionArgs a, Plan plan, uint32_t* err) {
  constexpr int kTile = kTileOf<kDim>;              // tokens of a page tile
  constexpr int kTailTile = kTile / 2;              // tokens of a tail tile
  constexpr int kMT = kTile / 16;                   // 16-token groups of a page tile
  constexpr int kKC = kDim / 64;                    // 64-channel column blocks of a key row
  constexpr int kVH = kDim == 256 ? 2 : 1;          // 128-channel halves of a value row
  constexpr int kVW = kDim == 64 ? 2 : 4;           // words of codes a lane loads of a value row's half
  constexpr int kOT = kDim / 16;                    // output tiles
  constexpr int kParts = 2;                         // fp16 parts of a weight in the paged tiles
  constexpr int kTailParts = kBf16 ? 3 : 2;         // parts of the tails' type in the tails
  // Outputs and sums are held in this unit, so that the largest weight counts as 1: a bf16 value
  // may be anything below 2^128, and 2^14 of it would pass float32.
  constexpr float kUnit = kBf16 ? 0x1p-14f : 1.f;
  constexpr int kTailRows = kTailTile / 8;          // token rows of a score tile that a tail tile fills
  __shared__ float4 s_o[kNT * kOT][kWarps][32];     // outputs of the CTA's warps where they share a segment
  __shared__ float s_m[kWarps][kNT * 8], s_l[kWarps][kNT * 8];
  const KittyKv8Cache& c = a.cache;
  const int lane = threadIdx.x & 31, lr = lane >> 2, lc = lane & 3;
  const int warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int D = kWhole ? kDim : c.head_dim, G = c.page_size, H = c.num_heads;
  const int g = a.num_q_heads / H;
  const int per_row = H * plan.passes, per_block = G / kTile;
  dev::wait_for_stream();
  asm volatile("griddepcontrol.launch_dependents;");   // merge_kernel may start to look where its parts will be
  const float fac16 = a.sm_scale * kLog2e;

  // this warp's slice [f, f_end)
  __shared__ Rows s_rows;
  const bool few = a.batch <= kFew;
  const int rows_each = (a.batch + kWarps * 32 - 1) / (kWarps * 32);
  FewRows few_rows;
  const int64_t total = (few ? scan_few<kTile>(a, plan, per_row, few_rows, err)
                             : scan_rows<kTile>(a, plan, per_row, rows_each, s_rows, err)) * per_row;
  const int64_t per_warp = quotient(total + plan.warps - 1, plan.warps);
  const int64_t f0 = warp * per_warp, f_end = min(total, f0 + per_warp);
  if (f0 >= f_end) return;
  if (warp == 0 && lane == 0) plan.notes[int64_t(a.batch) * per_row].units = per_warp;
  const Place at = few ? locate_few(per_row, few_rows, f0) : locate<kTile>(a, plan, per_row, rows_each, s_rows, f0);
  int b = at.b, seg = at.seg;
  int64_t begin = at.begin;

  while (begin < f_end) {
    const int len = tokens_of(a, plan, b);
    const Tiles tl = tiles_of<kTile>(c, plan, len);
    if (tl.all == 0) { ++b; continue; }             // (units are left, so a later row has some)
    const int slot = a.seq_map ? a.seq_map[b] : b;
    const int h = seg / plan.passes, q0 = (seg - h * plan.passes) * plan.pass_heads;
    const int heads = min(plan.pass_heads, g - q0);
    const int64_t end = begin + tl.units(), here = begin;
    // this warp's tiles of the segment
    const int t0 = int(max(f0 - here - kSetup, int64_t(0))), t1 = int(min(f_end, end) - here) - kSetup;
    const int row_b = b;
    const int64_t segment = int64_t(b) * per_row + seg;
    begin = end;
    if (++seg == per_row) { seg = 0; ++b; }
    if (t0 >= t1) continue;                         // only setup units

    // ---- the tiles' loads
    uint4 kr[kMT * 2 * kKC];                        // keys: codes [group][row lr, lr + 8][column block], tail rows
    uint32_t vr[kMT * kVH * 4 * kVW];               // values: codes [group][half][token][word], tail rows
    float ks = 0.f, vs = 0.f;
    bool ok = true;
    int page = 0, sub = t0 % per_block, block = t0 / per_block;
    const int last_block = (min(t1, tl.paged) - 1) / per_block;     // (not used without paged tiles)
    const int32_t* table = c.block_table + int64_t(slot) * c.bt_s_slot;
    int win0 = block;                               // the lanes hold 32 block-table entries from win0 on
    int win = t0 < tl.paged && win0 + lane <= last_block ? table[win0 + lane] : 0;
    const int64_t tail_base = (int64_t(slot) * H + h) * G * D;
    // page of `block`: page 0 and not ok if it is no page of the pool
    auto turn_page = [&]() {
      if (block >= win0 + 32) {
        win0 = block;
        win = win0 + lane <= last_block ? table[win0 + lane] : 0;
      }
      page = __shfl_sync(0xffffffffu, win, block - win0);
      ok = page >= 0 && page < c.pages;
      if (!ok) {
        if (lane == 0) dev::flag(err, kErrPage);
        page = 0;
      }
    };
    // Ask L2 for the page's next tiles, where it has more than one: the loads of a tile find the
    // following ones on their way.  32 x 32K tokens at G = 64 (two tiles) take 325 us with it and
    // 332 without, 16 x 131K at G = 128 (four) 664 and 707; asking for eight at once costs (G =
    // 256: 370 us, 327 with four), and so does asking for short sequences (8 x 8K: 35.2, 33.5).
    auto prefetch = [&]() {
      if (per_block > 1 && sub % kAhead == 0 && lane < 2) {
        const int64_t at = ((int64_t(page) * H + h) * G + sub * kTile) * D;
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                     :: "l"(static_cast<const uint8_t*>(lane ? c.value_codes : c.key_codes) + at),
                        "r"(min(kAhead, per_block - sub) * kTile * D));
      }
    };
    auto load_keys = [&]() {
      const uint8_t* p = static_cast<const uint8_t*>(c.key_codes) +
                         ((int64_t(page) * H + h) * G + sub * kTile + lr) * D + 16 * lc;
#pragma unroll
      for (int r = 0; r < kMT * 2; ++r)
#pragma unroll
        for (int jj = 0; jj < kKC; ++jj)
          kr[r * kKC + jj] = kWhole || 64 * jj + 16 * lc < D ? ld_stream(p + r * 8 * D + 64 * jj)
                                                             : make_uint4(0, 0, 0, 0);
      ks = c.key_scale[int64_t(page) * H + h];
    };
    auto load_tail_keys = [&](int t) {
      const int tok = (t - tl.paged) * kTailTile + lr;
      const uint16_t* p = static_cast<const uint16_t*>(c.tail_k) + tail_base + tok * D + 16 * lc;
#pragma unroll
      for (int r = 0; r < kTailRows; ++r)
#pragma unroll
        for (int jj = 0; jj < kKC; ++jj) {
          const bool there = tok + 8 * r < tl.tail && (kWhole || 64 * jj + 16 * lc < D);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            kr[(r * kKC + jj) * 2 + i] = there ? ld_stream(p + r * 8 * D + 64 * jj + 8 * i) : make_uint4(0, 0, 0, 0);
        }
    };
    auto load_values = [&]() {
      const uint8_t* p = static_cast<const uint8_t*>(c.value_codes) +
                         ((int64_t(page) * H + h) * G + sub * kTile + 2 * lc) * D + 4 * kVW * lr;
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int vh = 0; vh < kVH; ++vh)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint8_t* x = p + (mt * 16 + (k / 2) * 8 + k % 2) * D + 128 * vh;
            const bool there = kWhole || 128 * vh + 4 * kVW * lr < D;
            uint32_t* v = vr + ((mt * kVH + vh) * 4 + k) * kVW;
            if constexpr (kVW == 4) {
              const uint4 u = there ? ld_stream(x) : make_uint4(0, 0, 0, 0);
              v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
            } else {
              const uint2 u = there ? ld_stream2(x) : make_uint2(0, 0);
              v[0] = u.x; v[1] = u.y;
            }
          }
      vs = c.value_scale[int64_t(page) * H + h];
    };
    auto load_tail_values = [&](int t) {
      // rows behind the tail's end may hold anything: they read as zero
#pragma unroll
      for (int vh = 0; vh < kVH; ++vh)
#pragma unroll
        for (int k = 0; k < 2 * kTailRows; ++k) {
          const int row = (t - tl.paged) * kTailTile + 2 * lc + (k / 2) * 8 + k % 2;
          const bool there = row < tl.tail && (kWhole || 128 * vh + 4 * kVW * lr < D);
          const uint16_t* x = static_cast<const uint16_t*>(c.tail_v) + tail_base + row * D + 128 * vh + 4 * kVW * lr;
#pragma unroll
          for (int i = 0; i < kVW / 2; ++i) {
            const uint4 u = there ? ld_stream(x + 8 * i) : make_uint4(0, 0, 0, 0);
            uint32_t* v = vr + ((vh * 2 * kTailRows + k) * (kVW / 2) + i) * 4;
            v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
          }
        }
    };
    const int p1 = min(t1, tl.paged);               // tiles in pages end here
    if (t0 < p1) {
      turn_page();
      prefetch();
      load_keys();
      load_values();
    } else {
      load_tail_keys(t0);
      load_tail_values(t0);
    }

    // ---- q: lane (lr, lc) holds head lr's channels 64 jj + 16 lc + 0..15 of each column block
    const uint16_t* qrow[kNT];
    uint32_t qf[kNT][4 * kKC][2];
    float fac[kNT][2];                              // of the two columns (heads) whose scores this lane gets
    auto load_q = [&](int nt) {
#pragma unroll
      for (int jj = 0; jj < kKC; ++jj) {
        uint4 u = make_uint4(0, 0, 0, 0), v = u;
        const int ch = 64 * jj + 16 * lc;
        if (qrow[nt] && (kWhole || ch < D)) {
          u = *reinterpret_cast<const uint4*>(qrow[nt] + ch);
          v = *reinterpret_cast<const uint4*>(qrow[nt] + ch + 8);
        }
        const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) qf[nt][4 * jj + i / 2][i % 2] = w[i];
      }
    };
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int qh = nt * 8 + lr;
      qrow[nt] = qh < heads ? static_cast<const uint16_t*>(a.q) + row_b * a.q_s_seq + (h * g + q0 + qh) * a.q_s_head
                            : nullptr;
      load_q(nt);
      float scale = 1.f;                            // of head lr
      if constexpr (kBf16) {
        if (t0 < tl.paged) {
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < 8 * kKC; ++i) {
            const float2 x = dev::to_f2<true>(qf[nt][i / 2][i % 2]);
            top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // 2^(14 - exponent): the largest element lands in [2^14, 2^15); an all-zero or
          // infinite row keeps its values
          const int e = int(__float_as_uint(top) >> 23);
          const float up = e > 0 && e < 255 ? __uint_as_float(uint32_t(min(max(127 + 14 + 127 - e, 1), 254)) << 23) : 1.f;
          scale = 1.f / up;                         // a power of two: exact
#pragma unroll
          for (int i = 0; i < 8 * kKC; ++i) {
            const float2 x = dev::to_f2<true>(qf[nt][i / 2][i % 2]);
            qf[nt][i / 2][i % 2] = dev::from_f2<false>(x.x * up, x.y * up);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) fac[nt][j] = __shfl_sync(0xffffffffu, scale, (2 * lc + j) * 4) * fac16;
    }

    float o[kNT][kOT][4], base[kNT][2], l[kNT][2];   // base: the reference less kHead
    bool far = false;                               // some reference is beyond kFar
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int i = 0; i < kOT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      base[nt][0] = base[nt][1] = kUnset;
      l[nt][0] = l[nt][1] = 0.f;
    }

    // Weights of one tile: products s (token rows lr and lr + 8 of each group, two head
    // columns), times f a score, become 2^(score - base).  `there(group, row)`: whether the
    // token exists.
    auto weigh = [&](auto& s, int nt, float f0_, float f1_, auto there) {
      constexpr int kGroups = sizeof(s) / sizeof(s[0]);
      float x[kGroups][4], top = -INFINITY;
      auto relative = [&](bool rounded) {
#pragma unroll
        for (int k = 0; k < kGroups; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float f = i & 1 ? f1_ : f0_, b = base[nt][i & 1];
            const float y = rounded ? __fsub_rn(__fmul_rn(s[k][i], f), b) : fmaf(s[k][i], f, -b);
            x[k][i] = there(k, i / 2) ? y : -INFINITY;
            top = fmaxf(top, x[k][i]);
          }
      };
      relative(false);
      // A score far above the reference, or none yet; or a reference so far out that its
      // rounding (it is a rounded product) is more than the weights' range, where the products
      // have to be rounded alike.  (The maxima drop NaN, so a NaN score moves no reference: its
      // weight is NaN, and with it the output.)
      if (far || !__all_sync(0xffffffffu, top <= kHead + kSlack)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float best = -INFINITY;
#pragma unroll
          for (int k = 0; k < kGroups; ++k) {
            if (there(k, 0)) best = fmaxf(best, s[k][j] * (j ? f1_ : f0_));
            if (there(k, 1)) best = fmaxf(best, s[k][2 + j] * (j ? f1_ : f0_));
          }
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 4));
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 8));
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 16));
          const float now = fmaxf(base[nt][j], best - kHead), alpha = ex2(base[nt][j] - now);
          base[nt][j] = now;
          far |= fabsf(now) > kFar && now != kUnset;
          l[nt][j] *= alpha;
#pragma unroll
          for (int i = 0; i < kOT; ++i) {
            o[nt][i][j] *= alpha;
            o[nt][i][2 + j] *= alpha;
          }
        }
        far = __any_sync(0xffffffffu, far);
        if (far) relative(true);
        else relative(false);
      }
#pragma unroll
      for (int k = 0; k < kGroups; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[k][i] = ex2(x[k][i]);
    };

    for (int t = t0; t < p1; ++t) {
      // ------------------------------------------------------------ kTile tokens of a page
      float s[kNT][kMT][4];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) s[nt][mt][0] = s[nt][mt][1] = s[nt][mt][2] = s[nt][mt][3] = 0.f;
#pragma unroll
      for (int jj = 0; jj < kKC; ++jj)
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) {
          const uint4 u0 = kr[(2 * mt) * kKC + jj], u1 = kr[(2 * mt + 1) * kKC + jj];
          const uint32_t w0[4] = {u0.x, u0.y, u0.z, u0.w}, w1[4] = {u1.x, u1.y, u1.z, u1.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a0, a1, a2, a3;
            codes_to_half<kCode>(w0[i], a0, a2);
            codes_to_half<kCode>(w1[i], a1, a3);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
              mma<false>(s[nt][mt], a0, a1, a2, a3, qf[nt][4 * jj + i][0], qf[nt][4 * jj + i][1]);
          }
        }
      const float ks_now = ks, vs_now = vs;
      const bool ok_now = ok;
      if (t + 1 < p1) {
        if (++sub == per_block) {
          sub = 0;
          ++block;
          turn_page();
        }
        prefetch();
        load_keys();
      } else if (t + 1 < t1) {
        load_tail_keys(t + 1);
      }
      uint32_t wb[kNT][kMT][kParts][2];           // weights as the other operand: tokens 0..7 and 8..15 of a group
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        weigh(s[nt], nt, fac[nt][0] * ks_now, fac[nt][1] * ks_now, [&](int, int) { return ok_now; });
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t hi = dev::from_f2<false>(s[nt][mt][2 * r], s[nt][mt][2 * r + 1]);
            const float2 back = dev::to_f2<false>(hi);
            wb[nt][mt][0][r] = transpose8x8(hi);
            wb[nt][mt][1][r] =
                transpose8x8(dev::from_f2<false>(s[nt][mt][2 * r] - back.x, s[nt][mt][2 * r + 1] - back.y));
            l[nt][0] += s[nt][mt][2 * r];
            l[nt][1] += s[nt][mt][2 * r + 1];
          }
      }
      float vmul = vs_now * kUnit;
      if (!ok_now) {                              // page 0 stood in for it: its codes may be NaN, which no weight of 0 takes away
        vmul = 0.f;
#pragma unroll
        for (int i = 0; i < kMT * kVH * 4 * kVW; ++i) vr[i] = 0u;
      }
#pragma unroll
      for (int vh = 0; vh < kVH; ++vh)
#pragma unroll
        for (int x = 0; x < kVW; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {           // bytes 0, 1 or 2, 3 of the word: two channels
            const uint32_t sel = y ? 0x7362u : 0x5140u;
            const int i = (vh * kVW + x) * 2 + y;
            float acc[kNT][4];
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
            for (int mt = 0; mt < kMT; ++mt) {
              const uint32_t* v = vr + (mt * kVH + vh) * 4 * kVW + x;
              uint32_t a0, a1, a2, a3;
              codes_to_half<kCode>(prmt(v[0], v[kVW], sel), a0, a1);
              codes_to_half<kCode>(prmt(v[2 * kVW], v[3 * kVW], sel), a2, a3);
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                for (int p = 0; p < kParts; ++p)
                  mma<false>(acc[nt], a0, a1, a2, a3, wb[nt][mt][p][0], wb[nt][mt][p][1]);
            }
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][i][e] = fmaf(acc[nt][e], vmul, o[nt][i][e]);
          }
      if (t + 1 < p1) load_values();
      else if (t + 1 < t1) load_tail_values(t + 1);
    }
    if constexpr (kBf16) {                          // bf16 products in the tail: q as it is
      if (t0 < p1 && p1 < t1) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) load_q(nt);
      }
    }
    for (int t = max(t0, p1); t < t1; ++t) {
      // ------------------------------------------------------------ kTailTile tokens of 16 bits
      const int tok = (t - tl.paged) * kTailTile + lr;
      float s[kNT][1][4];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) s[nt][0][0] = s[nt][0][1] = s[nt][0][2] = s[nt][0][3] = 0.f;
#pragma unroll
      for (int jj = 0; jj < kKC; ++jj)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 u0 = kr[jj * 2 + i];
          const uint4 u1 = kTailRows == 2 ? kr[((kTailRows - 1) * kKC + jj) * 2 + i] : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            mma<kBf16>(s[nt][0], u0.x, u1.x, u0.y, u1.y, qf[nt][4 * jj + 2 * i][0], qf[nt][4 * jj + 2 * i][1]);
            mma<kBf16>(s[nt][0], u0.z, u1.z, u0.w, u1.w, qf[nt][4 * jj + 2 * i + 1][0], qf[nt][4 * jj + 2 * i + 1][1]);
          }
        }
      if (t + 1 < t1) load_tail_keys(t + 1);
      uint32_t wb[kNT][kTailParts][2];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        weigh(s[nt], nt, fac16, fac16, [&](int, int row) { return row < kTailRows && tok + 8 * row < tl.tail; });
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float2 left = make_float2(s[nt][0][2 * r] * kUnit, s[nt][0][2 * r + 1] * kUnit);
#pragma unroll
          for (int p = 0; p < kTailParts; ++p) {  // each takes what the ones before leave
            const uint32_t part = dev::from_f2<kBf16>(left.x, left.y);
            const float2 back = dev::to_f2<kBf16>(part);
            wb[nt][p][r] = transpose8x8(part);
            left = make_float2(left.x - back.x, left.y - back.y);
          }
        }
        l[nt][0] += s[nt][0][0] + s[nt][0][2];
        l[nt][1] += s[nt][0][1] + s[nt][0][3];
      }
#pragma unroll
      for (int vh = 0; vh < kVH; ++vh)
#pragma unroll
        for (int x = 0; x < 2 * kVW; ++x) {       // a word holds the channel pair of one output tile
          const int i = vh * kVW * 2 + x;
          const uint32_t* v = vr + vh * 2 * kTailRows * 2 * kVW + x;
          const uint32_t a0 = prmt(v[0], v[2 * kVW], 0x5410), a1 = prmt(v[0], v[2 * kVW], 0x7632);
          const uint32_t w2 = kTailRows == 2 ? v[(kTailRows - 1) * 4 * kVW] : 0u;
          const uint32_t w3 = kTailRows == 2 ? v[(kTailRows - 1) * 6 * kVW] : 0u;
          const uint32_t a2 = prmt(w2, w3, 0x5410), a3 = prmt(w2, w3, 0x7632);
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
            for (int p = 0; p < kTailParts; ++p) mma<kBf16>(o[nt][i], a0, a1, a2, a3, wb[nt][p][0], wb[nt][p][1]);
          }
        }
      if (t + 1 < t1) load_tail_values(t + 1);
    }

    // ---- store: the segment's output, or this warp's or CTA's part of it
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
        l[nt][j] *= kUnit;
      }
    const bool all_here = t0 == 0 && t1 == tl.all;
    if (t0 == 0 && lane == 0) plan.notes[segment] = all_here ? Note{0, -1} : Note{here, end - here};
    const bool together = cta_inside(blockIdx.x, per_warp, here, end);
    int x0 = 0, x1 = kOT / 2;                       // pairs of output tiles that this warp stores
    const int w = threadIdx.x >> 5;
    if (together) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
        for (int i = 0; i < kOT; ++i)
          s_o[nt * kOT + i][w][lane] = make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]);
        if (lr == 0) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s_m[w][nt * 8 + 2 * lc + j] = base[nt][j];
            s_l[w][nt * 8 + 2 * lc + j] = l[nt][j];
          }
        }
      }
      __syncthreads();                              // (each CTA comes here at most once: its slices lie in the segment)
      constexpr int kEach = (kOT / 2 + kWarps - 1) / kWarps;
      x0 = w * kEach;
      x1 = min(x0 + kEach, kOT / 2);
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        float k[kWarps][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int col = nt * 8 + 2 * lc + j;
          float top = s_m[0][col];
#pragma unroll
          for (int i = 1; i < kWarps; ++i) top = fmaxf(top, s_m[i][col]);
          base[nt][j] = top;
          l[nt][j] = 0.f;
#pragma unroll
          for (int i = 0; i < kWarps; ++i) {
            k[i][j] = ex2(s_m[i][col] - top);
            l[nt][j] = fmaf(k[i][j], s_l[i][col], l[nt][j]);
          }
        }
#pragma unroll
        for (int i = 0; i < kOT; ++i) {
          if (i / 2 < x0 || i / 2 >= x1) continue;
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int q = 0; q < kWarps; ++q) {
            const float4 v = s_o[nt * kOT + i][q][lane];
            sum.x = fmaf(k[q][0], v.x, sum.x);
            sum.y = fmaf(k[q][1], v.y, sum.y);
            sum.z = fmaf(k[q][0], v.z, sum.z);
            sum.w = fmaf(k[q][1], v.w, sum.w);
          }
          o[nt][i][0] = sum.x; o[nt][i][1] = sum.y; o[nt][i][2] = sum.z; o[nt][i][3] = sum.w;
        }
      }
    }
    // the slice's first segment, or its last; of a CTA's warps together, the first's place
    const int64_t place = together ? 2 * int64_t(blockIdx.x) * kWarps : 2 * int64_t(warp) + (here > f0);
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int qh = nt * 8 + 2 * lc + j;
        if (qh >= heads) continue;
        const float inv = l[nt][j] == 0.f ? 0.f : 1.f / l[nt][j];
        uint16_t* out = static_cast<uint16_t*>(a.out) + row_b * a.out_s_seq + (h * g + q0 + qh) * a.out_s_head;
        float* part = plan.part_o + (place * plan.pass_heads + qh) * D;
        if (!all_here && lr == 0 && x0 == 0) {
          float* ml = plan.part_ml + (place * plan.pass_heads + qh) * 2;
          ml[0] = base[nt][j];
          ml[1] = l[nt][j];
        }
#pragma unroll
        for (int x = 0; x < kOT / 2; ++x) {         // four channels from two output tiles
          if (x < x0 || x >= x1) continue;
          const int vh = x / kVW, ch = 128 * vh + 4 * kVW * lr + 4 * (x % kVW);
          if (!kWhole && ch >= D) continue;
          const float v0 = o[nt][2 * x][j], v1 = o[nt][2 * x][2 + j], v2 = o[nt][2 * x + 1][j], v3 = o[nt][2 * x + 1][2 + j];
          if (all_here)
            *reinterpret_cast<uint2*>(out + ch) =
                make_uint2(dev::from_f2<kBf16>(v0 * inv, v1 * inv), dev::from_f2<kBf16>(v2 * inv, v3 * inv));
          else
            *reinterpret_cast<float4*>(part + ch) = make_float4(v0, v1, v2, v3);
        }
      }
  }
}

// Joins the parts of a segment: out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i; zeros for an
// empty slot.  Where segments are few, each has many parts: the team is a CTA for one query
// head, whose threads form groups of one thread for each 16-byte vector of the head; the
// groups take the parts in turn, each with its own reference, and are joined in order.
// Otherwise the team is a warp, for `heads_each` heads.
template <int kTile, bool kBf16, int kTeam>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(KittyKv8AttentionArgs a, Plan plan, int heads_each) {
  constexpr int kBatch = kTeam == 32 ? 4 : 8;          // parts whose loads are in flight
  __shared__ float4 s_sum[kTeam == 32 ? 1 : kTeam];
  __shared__ float s_l[kTeam == 32 ? 1 : kTeam], s_m[kTeam == 32 ? 1 : kTeam];
  const KittyKv8Cache& c = a.cache;
  const int tid = threadIdx.x % kTeam;
  const int D = c.head_dim, g = a.num_q_heads / c.num_heads, per_row = c.num_heads * plan.passes;
  const uint32_t team = blockIdx.x * (kMergeThreads / kTeam) + threadIdx.x / kTeam;
  const uint32_t per_segment = (plan.pass_heads + heads_each - 1) / heads_each, segment = team / per_segment;
  const int b = int(segment / per_row), seg = int(segment - uint32_t(b) * per_row);
  const int h = seg / plan.passes, q0 = (seg - h * plan.passes) * plan.pass_heads;
  const int first = int(team - segment * per_segment) * heads_each;
  const int heads = min(min(plan.pass_heads, g - q0) - first, heads_each);
  Note note{0, -2};
  int64_t per_warp = 1;
  // Where the segment begins, while attention_kernel still runs: one sequence of 4096 tokens takes
  // 9.3 us so and 9.9 with the note, 48 segments 18.3 and 18.8.  (Up to two rows a lane, which is
  // all that segments for CTAs come to at 128 and 256 channels.)
  if (kTeam != 32 && a.batch <= 64) {
    int64_t before = 0, total = 0;
    for (int i = threadIdx.x & 31; i < a.batch; i += 32) {
      const int64_t n = units_of_row<kTile, true>(a, plan, i);
      total += n;
      if (i < b) before += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    per_warp = max(quotient(total * per_row + plan.warps - 1, plan.warps), int64_t(1));
    note.units = units_of_row<kTile, true>(a, plan, b);
    note.begin = before * per_row + int64_t(seg) * note.units;
  }
  dev::wait_for_stream();                              // attention_kernel is done and its parts are visible
  if (b >= a.batch || heads <= 0) return;
  if (note.units == -2) {
    note = plan.notes[segment];
    per_warp = plan.notes[int64_t(a.batch) * per_row].units;
  }
  if (note.units < 0) return;                          // stored by its warp
  uint16_t* out = static_cast<uint16_t*>(a.out) + b * a.out_s_seq + int64_t(h * g + q0 + first) * a.out_s_head;
  const int vecs = D / 4, work = heads * vecs;         // (vecs at most 64)
  if (note.units == 0) {
    for (int u = tid; u < work; u += kTeam)
      *reinterpret_cast<uint2*>(out + (u / vecs) * a.out_s_head + (u % vecs) * 4) = make_uint2(0, 0);
    return;
  }
  const int64_t begin = note.begin, end = begin + note.units, per_cta = per_warp * kWarps;
  const int w0 = int(quotient(begin + kSetup, per_warp)), w1 = int(quotient(end - 1, per_warp));
  if (w0 == w1) return;                                // stored by its warp
  // its parts: warps w0 .., whole CTAs c0 .. c1 - 1, warps .. w1
  const int c0 = int(quotient(begin + kSetup + per_cta - 1, per_cta)), c1 = int(quotient(end, per_cta));
  const int n2 = max(c1 - c0, 0);
  const int n1 = n2 ? c0 * kWarps - w0 : w1 - w0 + 1;
  const int parts = n2 ? n1 + n2 + (w1 - c1 * kWarps + 1) : n1;
  auto place = [&](int i) {
    const int w = i < n1 ? w0 + i : i < n1 + n2 ? (c0 + i - n1) * kWarps : c1 * kWarps + (i - n1 - n2);
    return (2 * int64_t(w) + (begin > w * per_warp)) * plan.pass_heads + first;
  };
  const int groups = kTeam == 32 ? 1 : kTeam / vecs;
  for (int u0 = 0; u0 < work; u0 += kTeam) {           // (a CTA: one round)
    const int group = kTeam == 32 ? 0 : tid / vecs, u = kTeam == 32 ? u0 + tid : tid - group * vecs;
    const int head = kTeam == 32 ? u / vecs : 0, v = u - head * vecs;
    const bool mine = u < work && group < groups;
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = group; mine && i0 < parts; i0 += groups * kBatch) {
      float2 ml[kBatch];
      float4 p[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int i = i0 + k * groups;
        ml[k] = make_float2(-INFINITY, 0.f);
        p[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < parts) {
          const int64_t at = place(i) + head;
          ml[k] = *reinterpret_cast<const float2*>(plan.part_ml + at * 2);
          p[k] = *reinterpret_cast<const float4*>(plan.part_o + at * D + v * 4);
        }
      }
      const float old = top;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) top = fmaxf(top, ml[k].x);
      const float ref = top == -INFINITY ? 0.f : top, f0 = ex2(old - ref);
      sum *= f0;
      acc = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const float f = ex2(ml[k].x - ref);
        sum = fmaf(f, ml[k].y, sum);
        acc.x = fmaf(f, p[k].x, acc.x);
        acc.y = fmaf(f, p[k].y, acc.y);
        acc.z = fmaf(f, p[k].z, acc.z);
        acc.w = fmaf(f, p[k].w, acc.w);
      }
    }
    if constexpr (kTeam != 32) {
      s_sum[tid] = acc;
      s_l[tid] = sum;
      s_m[tid] = top;
      __syncthreads();
      if (mine && group == 0) {
        for (int k = 1; k < groups; ++k) top = fmaxf(top, s_m[k * vecs + v]);
        const float ref = top == -INFINITY ? 0.f : top;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
        sum = 0.f;
        for (int k = 0; k < groups; ++k) {
          const float f = ex2(s_m[k * vecs + v] - ref);
          const float4 p = s_sum[k * vecs + v];
          sum = fmaf(f, s_l[k * vecs + v], sum);
          acc.x = fmaf(f, p.x, acc.x);
          acc.y = fmaf(f, p.y, acc.y);
          acc.z = fmaf(f, p.z, acc.z);
          acc.w = fmaf(f, p.w, acc.w);
        }
      }
    }
    if (mine && group == 0) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint2*>(out + head * a.out_s_head + v * 4) =
          make_uint2(dev::from_f2<kBf16>(acc.x * inv, acc.y * inv), dev::from_f2<kBf16>(acc.z * inv, acc.w * inv));
    }
  }
}

// merge_kernel starts while attention_kernel runs and waits in front of the first part.
template <int kTile, bool kBf16, int kTeam>
int launch_merge(const KittyKv8AttentionArgs& a, const Plan& plan, int heads_each, cudaStream_t s) {
  const unsigned teams =
      unsigned(a.batch) * a.cache.num_heads * plan.passes * ((plan.pass_heads + heads_each - 1) / heads_each);
  const dim3 grid((teams + kMergeThreads / kTeam - 1) / (kMergeThreads / kTeam));
  return launch_dependent("kv8_attention (merge)", merge_kernel<kTile, kBf16, kTeam>, grid, kMergeThreads, 0, s, a, plan,
                          heads_each);
}

// Resident CTAs per SM that a kernel's registers allow (asked once per kernel).
template <int kDim, int kNT, bool kWhole, bool kBf16, int kCode>
int resident() {
  static std::atomic<int> known{0};
  if (known.load(std::memory_order_relaxed) == 0) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attention_kernel<kDim, kNT, kWhole, kBf16, kCode>,
                                                      kWarps * 32, 0) != cudaSuccess || n < 1) {
      cudaGetLastError();
      return 1;
    }
    known.store(n, std::memory_order_relaxed);
  }
  return known.load(std::memory_order_relaxed);
}

// The workspace: the segments' notes, the parts' references and sums, and
// their outputs, each from a 256-byte boundary.  Returns its bytes.
size_t lay_out(Plan& plan, const KittyKv8AttentionArgs& a, uint8_t* base) {
  const auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t segments = size_t(a.batch) * a.cache.num_heads * plan.passes;
  const size_t parts = size_t(2) * plan.warps * plan.pass_heads;
  const size_t begins = up((segments + 1) * sizeof(Note)), ml = up(parts * 8);
  plan.notes = reinterpret_cast<Note*>(base);
  plan.part_ml = reinterpret_cast<float*>(base + begins);
  plan.part_o = reinterpret_cast<float*>(base + begins + ml);
  return begins + ml + parts * a.cache.head_dim * 4;
}

template <int kDim, int kNT, bool kWhole, bool kBf16, int kCode>
int launch(const KittyKv8AttentionArgs& a, Plan plan, uint32_t* err, cudaStream_t s, size_t* bytes) {
  const int grid = sm_count() * resident<kDim, kNT, kWhole, kBf16, kCode>();
  plan.warps = grid * kWarps;
  const size_t need = lay_out(plan, a, static_cast<uint8_t*>(a.workspace));
  if (bytes) { *bytes = need; return KITTY_OK; }
  if (a.workspace_bytes < need)
    return fail(KITTY_ERR_WORKSPACE, "kv8_attention", "workspace smaller than kitty_kv8_attention_workspace_size()");
  const int rc = launch_dependent("kv8_attention", attention_kernel<kDim, kNT, kWhole, kBf16, kCode>, dim3(unsigned(grid)),
                                  kWarps * 32, 0, s, a, plan, err);
  if (rc != KITTY_OK) return rc;
  // Many warps to a segment: a CTA joins a head (128 channels, 8192 tokens each: 48 segments take
  // 25.9 us so and 29.8 with warps).  The two meet at 76 segments whatever the channels, which is
  // where the rule changes at 64; at 128 channels 56 to 72 segments, and at 256 from 40 on, would
  // still be 2 to 7 us faster with CTAs.  Otherwise a warp joins as many heads as it has lanes
  // for: 256 mixed lengths, 2048 segments of 5 heads, take 57.0 us all told (one head a warp
  // 58.8, all five 59.2).
  const int64_t segments = int64_t(a.batch) * a.cache.num_heads * plan.passes;
  const int heads_each = std::min(std::max(1, 128 / a.cache.head_dim), plan.pass_heads);
  return segments * 32 < plan.warps ? launch_merge<kTileOf<kDim>, kBf16, kMergeThreads>(a, plan, 1, s)
                                    : launch_merge<kTileOf<kDim>, kBf16, 32>(a, plan, heads_each, s);
}

template <int kDim, bool kWhole, bool kBf16, int kCode>
int launch_heads(const KittyKv8AttentionArgs& a, uint32_t* err, cudaStream_t s, size_t* bytes) {
  // Query heads of a KV head in passes of 8 or 16: 16 columns share every conversion of
  // a code, but at 256 channels their outputs would not fit the registers.
  const int g = a.num_q_heads / a.cache.num_heads;
  constexpr bool kTwo = kDim <= 128;
  Plan plan{};
  const uint32_t k = uint32_t(a.cache.page_size) / 32;
  plan.per_page = (0x80000000u + k - 1) / k;
  const int most = kTwo && g > 8 ? 16 : 8;
  plan.passes = (g + most - 1) / most;
  plan.pass_heads = (g + plan.passes - 1) / plan.passes;
  if constexpr (kTwo) {
    if (plan.pass_heads > 8) return launch<kDim, 2, kWhole, kBf16, kCode>(a, plan, err, s, bytes);
  }
  return launch<kDim, 1, kWhole, kBf16, kCode>(a, plan, err, s, bytes);
}

template <bool kBf16, int kCode>
int launch_dim(const KittyKv8AttentionArgs& a, uint32_t* err, cudaStream_t s, size_t* bytes) {
  const int D = a.cache.head_dim;
  if (D == 64) return launch_heads<64, true, kBf16, kCode>(a, err, s, bytes);
  if (D < 64) return launch_heads<64, false, kBf16, kCode>(a, err, s, bytes);
  if (D == 128) return launch_heads<128, true, kBf16, kCode>(a, err, s, bytes);
  if (D < 128) return launch_heads<128, false, kBf16, kCode>(a, err, s, bytes);
  if (D == 256) return launch_heads<256, true, kBf16, kCode>(a, err, s, bytes);
  return launch_heads<256, false, kBf16, kCode>(a, err, s, bytes);
}

int dispatch(const KittyKv8AttentionArgs& a, uint32_t* err, cudaStream_t s, size_t* bytes) {
  if (a.cache.dtype == KITTY_KV8_BF16)
    return a.cache.code == KITTY_KV8_E4M3 ? launch_dim<true, KITTY_KV8_E4M3>(a, err, s, bytes)
                                          : launch_dim<true, KITTY_KV8_INT8>(a, err, s, bytes);
  return a.cache.code == KITTY_KV8_E4M3 ? launch_dim<false, KITTY_KV8_E4M3>(a, err, s, bytes)
                                        : launch_dim<false, KITTY_KV8_INT8>(a, err, s, bytes);
}

int check_attention(const KittyKv8AttentionArgs* a, const char* what) {
  if (!a) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "args is NULL");
  const int rc = check_cache(&a->cache, what);
  if (rc != KITTY_OK) return rc;
  if (a->batch < 0 || a->num_q_heads <= 0) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "negative or zero size");
  if (a->num_q_heads % a->cache.num_heads)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "num_q_heads must be a multiple of num_heads");
  if (!a->seq_map && a->batch > a->cache.slots)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "more queries than slots");
  if (int64_t(a->batch) * a->num_q_heads > 0x3fffffffLL)   // (passes round a KV head's query heads up, to less than twice)
    return fail(KITTY_ERR_UNSUPPORTED, what, "batch * num_q_heads must fit 30 bits");
  return KITTY_OK;
}

}  // namespace
}  // namespace kitty8

using namespace kitty8;

extern "C" int kitty_kv8_attention_workspace_size(const KittyKv8AttentionArgs* a, size_t* bytes) {
  const char* what = "kv8_attention_workspace_size";
  const int rc = check_attention(a, what);
  if (rc != KITTY_OK) return rc;
  if (!bytes) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "bytes is NULL");
  return dispatch(*a, nullptr, nullptr, bytes);
}

extern "C" int kitty_kv8_attention(const KittyKv8AttentionArgs* a, void* stream) {
  const char* what = "kv8_attention";
  const int rc = check_attention(a, what);
  if (rc != KITTY_OK) return rc;
  if (a->batch == 0) return KITTY_OK;
  if (!a->q || !a->out) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "NULL q or out");
  if (!aligned(a->q, 16) || a->q_s_seq % 8 || a->q_s_head % 8)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "q rows must be 16-byte aligned (strides multiples of 8 elements)");
  if (!aligned(a->out, 8) || a->out_s_seq % 4 || a->out_s_head % 4)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "out rows must be 8-byte aligned (strides multiples of 4 elements)");
  if (!a->workspace || !aligned(a->workspace, 16))
    return fail(KITTY_ERR_WORKSPACE, what, "workspace missing or not 16-byte aligned");
  uint32_t* err = error_word();
  if (!err) return fail(KITTY_ERR_CUDA, what, "no CUDA device");
  KittyKv8AttentionArgs args = *a;
  if (args.cache.pages == 0) args.cache.max_pages = 0;     // without a page 0 to stand for a missing one, tails only
  return dispatch(args, err, as_stream(stream), nullptr);
}
