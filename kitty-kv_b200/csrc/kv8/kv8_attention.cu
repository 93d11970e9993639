// Decode attention over the 8-bit paged cache.
//
// Per (slot, KV head, pass of up to 8 kNT query heads) - a segment - with scores in
// base 2: s_t = sm_scale log2(e) key_scale (q . code_t), and a running maximum m,
//   l <- l 2^(m - m') + sum_t 2^(s_t - m'),   O <- O 2^(m - m') + value_scale sum_t 2^(s_t - m') code_t.
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
// keeps elements down to 2^-29 of it exact.  Weights are rounded to fp16 with 2^14 of
// headroom; for fp16 outputs, whose own rounding is as small, they are split in two
// parts (16-bit tails of bf16 slots: two bf16 parts).
//
// All segments' tiles (kTile tokens of a page, 16 of a tail) are laid end to end and every
// warp of a fixed grid takes one contiguous slice; warps never wait for one another.  The
// next tile's keys are requested when this tile's scores are done, its values when this
// tile's output is.  A segment inside one slice is stored at once; the parts of one that
// crosses slices go to the workspace (two places a warp) and are joined by merge_kernel.
#include "kv8_common.cuh"

namespace kitty8 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHead = 14.f;          // weights are kept times 2^kHead, so that small ones stay normal in fp16
constexpr int kWarps = 4;              // per CTA
constexpr int kMergeThreads = 256;

struct Plan {
  int passes, pass_heads;              // query heads of a KV head in passes of pass_heads
  int warps;                           // of the whole grid
  float* part_ml;                      // [2 warps][pass_heads][2]  maximum, sum
  float* part_o;                       // [2 warps][pass_heads][D]
};

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream2(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
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

// Tiles of a slot's segments: its whole pages, then its tail.
struct Tiles {
  int paged, all, tail;                // tiles in pages, all tiles, tail tokens
};
template <int kTile>
__device__ __forceinline__ Tiles tiles_of(const KittyKv8Cache& c, int len) {
  const int blocks = min(len / c.page_size, c.max_pages), tail = len % c.page_size;
  const int paged = blocks * (c.page_size / kTile);
  return Tiles{paged, paged + (tail + 15) / 16, tail};
}
__device__ __forceinline__ int slot_of(const KittyKv8AttentionArgs& a, int b, uint32_t* err) {
  const int s = a.seq_map ? a.seq_map[b] : b;
  if (s >= 0 && s < a.cache.slots) return s;
  if (err) dev::flag(err, kErrSlot);
  return -1;
}
// Tokens of batch row b: 0 where its slot or its length is out of range.
__device__ __forceinline__ int tokens_of(const KittyKv8AttentionArgs& a, int b, uint32_t* err = nullptr) {
  const int s = slot_of(a, b, err);
  if (s < 0) return 0;
  const int len = a.cache.lengths[s];
  if (len >= 0 && len / a.cache.page_size <= a.cache.max_pages) return len;
  if (err) dev::flag(err, kErrLength);
  return 0;
}

struct Place {
  int64_t total;       // tiles of the whole batch
  int64_t begin;       // first tile of the segment found
  int b, seg;          // its batch row; its index among the row's segments; b < 0: none
};

// By the whole warp: all tiles, and the segment that holds tile f.  Row b has
// `per_row` = H * passes segments of equal length.
template <int kTile>
__device__ __forceinline__ Place locate(const KittyKv8AttentionArgs& a, int per_row, int64_t f) {
  const int lane = threadIdx.x & 31;
  Place r{0, 0, -1, 0};
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    const int one = b < a.batch ? tiles_of<kTile>(a.cache, tokens_of(a, b)).all : 0;
    const int64_t mine = int64_t(one) * per_row;
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const int64_t start = r.total + incl - mine;
    const uint32_t hit = __ballot_sync(0xffffffffu, f >= start && f < start + mine);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int64_t at = __shfl_sync(0xffffffffu, start, src);
      const int len = __shfl_sync(0xffffffffu, one, src);
      r.b = b0 + src;
      r.seg = int((f - at) / len);
      r.begin = at + int64_t(r.seg) * len;
    }
    r.total += __shfl_sync(0xffffffffu, incl, 31);
  }
  return r;
}

// kDim: 64, 128 or 256 channels in registers; kWhole: head_dim == kDim (else the missing
// channels read as zero).  kNT: tiles of 8 query heads.
template <int kDim, int kNT, bool kWhole, bool kBf16, int kCode>
__global__ void __launch_bounds__(kWarps * 32) attention_kernel(KittyKv8AttentionArgs a, Plan plan, uint32_t* err) {
  constexpr int kTile = kDim == 256 ? 16 : 32;      // tokens of a page tile
  constexpr int kMT = kTile / 16;                   // 16-token groups of it
  constexpr int kKC = kDim / 64;                    // 64-channel column blocks of a key row
  constexpr int kVH = kDim == 256 ? 2 : 1;          // 128-channel halves of a value row
  constexpr int kVW = kDim == 64 ? 2 : 4;           // words of codes a lane loads of a value row's half
  constexpr int kOT = kDim / 16;                    // output tiles
  constexpr int kParts = kBf16 ? 1 : 2;             // fp16 parts of a weight in the paged tiles
  const KittyKv8Cache& c = a.cache;
  const int lane = threadIdx.x & 31, lr = lane >> 2, lc = lane & 3;
  const int warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int D = kWhole ? kDim : c.head_dim, G = c.page_size, H = c.num_heads;
  const int g = a.num_q_heads / H;
  const int per_row = H * plan.passes;

  // this warp's slice [f, f_end)
  if (warp == 0)
    for (int b = lane; b < a.batch; b += 32) tokens_of(a, b, err);
  Place at = locate<kTile>(a, per_row, -1);
  const int64_t per_warp = (at.total + plan.warps - 1) / plan.warps;
  int64_t f = warp * per_warp;
  const int64_t f_end = min(at.total, f + per_warp);
  if (f >= f_end) return;
  at = locate<kTile>(a, per_row, f);
  int b = at.b, seg = at.seg;
  int64_t begin = at.begin;

  while (f < f_end) {
    const int len = tokens_of(a, b);
    const Tiles tl = tiles_of<kTile>(c, len);
    if (tl.all == 0) { ++b; seg = 0; continue; }    // (f < total: a later row has tiles)
    const int slot = a.seq_map ? a.seq_map[b] : b;
    const int h = seg / plan.passes, q0 = (seg % plan.passes) * plan.pass_heads;
    const int heads = min(plan.pass_heads, g - q0);
    const int64_t seg_end = begin + tl.all;
    const int t0 = int(f - begin), t1 = int(min(f_end, seg_end) - begin);   // this warp's tiles of the segment
    const int p1 = min(t1, tl.paged);               // its tiles in pages end here

    // q: lane (lr, lc) holds head lr's channels 64 jj + 16 lc + 0..15 of each column block
    const uint16_t* qrow[kNT];
    uint32_t qf[kNT][4 * kKC][2];
    float fac[kNT][2];                              // of the two columns (heads) whose scores this lane gets
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int qh = nt * 8 + lr;
      qrow[nt] = qh < heads ? static_cast<const uint16_t*>(a.q) + b * a.q_s_seq + (h * g + q0 + qh) * a.q_s_head : nullptr;
      float top = 0.f;
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
        for (int i = 0; i < 8; ++i) {
          qf[nt][4 * jj + i / 2][i % 2] = w[i];
          if constexpr (kBf16) {
            const float2 x = dev::to_f2<true>(w[i]);
            top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
          }
        }
      }
      float scale = 1.f;                            // of head lr
      if constexpr (kBf16) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^(14 - exponent): the largest element lands in [2^14, 2^15); an all-zero or
        // infinite row keeps its values
        const int e = int(__float_as_uint(top) >> 23);
        const float up = e > 0 && e < 255 ? __uint_as_float(uint32_t(min(max(127 + 14 + 127 - e, 1), 254)) << 23) : 1.f;
        scale = 1.f / up;                           // a power of two (or its subnormal neighbour's inverse): exact
#pragma unroll
        for (int i = 0; i < 4 * kKC; ++i) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 x = dev::to_f2<true>(qf[nt][i][k]);
            qf[nt][i][k] = dev::from_f2<false>(x.x * up, x.y * up);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
        fac[nt][j] = __shfl_sync(0xffffffffu, scale, (2 * lc + j) * 4) * (a.sm_scale * kLog2e);
    }

    float o[kNT][kOT][4], m[kNT][2], l[kNT][2];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int i = 0; i < kOT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    // Softmax step of one tile: scores s (token rows lr and lr + 8 of each group, two head
    // columns) become weights 2^(s - m + kHead), the sums are brought up to date and
    // alpha gets the factor of what was there before.
    auto softmax = [&](auto& s, int nt, float (&alpha)[2]) {
      constexpr int kGroups = sizeof(s) / sizeof(s[0]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float top = m[nt][j];
#pragma unroll
        for (int k = 0; k < kGroups; ++k) top = fmaxf(top, fmaxf(s[k][j], s[k][2 + j]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const float ref = top == -INFINITY ? 0.f : top;      // nothing yet: all weights 0
        alpha[j] = ex2(m[nt][j] - ref);
        m[nt][j] = top;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          s[k][j] = ex2(s[k][j] - (ref - kHead));
          s[k][2 + j] = ex2(s[k][2 + j] - (ref - kHead));
        }
      }
    };

    // ------------------------------------------------------------------ pages
    if (t0 < p1) {
      const int per_block = G / kTile;
      const int32_t* table = c.block_table + int64_t(slot) * c.bt_s_slot;
      int win0 = t0 / per_block;                    // the lanes hold 32 block-table entries from win0 on
      const int last_block = (p1 - 1) / per_block;
      int win = win0 + lane <= last_block ? table[win0 + lane] : 0;
      // block of a tile -> page (0 and not ok if it is no page of the pool)
      auto page_at = [&](int block, bool& ok) {
        if (block >= win0 + 32) {
          win0 = block;
          win = win0 + lane <= last_block ? table[win0 + lane] : 0;
        }
        const int p = __shfl_sync(0xffffffffu, win, block - win0);
        ok = p >= 0 && p < c.pages;
        if (!ok && lane == 0) dev::flag(err, kErrPage);
        return ok ? p : 0;
      };
      uint4 kr[kMT][2][kKC];
      uint32_t vr[kMT][kVH][4][kVW];
      float ks, vs;
      auto load_keys = [&](int page, int sub) {
        const uint8_t* p = static_cast<const uint8_t*>(c.key_codes) +
                           ((int64_t(page) * H + h) * G + sub * kTile + lr) * D + 16 * lc;
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int jj = 0; jj < kKC; ++jj)
              kr[mt][r][jj] = kWhole || 64 * jj + 16 * lc < D ? ld_stream(p + (mt * 16 + r * 8) * D + 64 * jj)
                                                              : make_uint4(0, 0, 0, 0);
        ks = __ldg(c.key_scale + int64_t(page) * H + h);
      };
      auto load_values = [&](int page, int sub) {
        const uint8_t* p = static_cast<const uint8_t*>(c.value_codes) +
                           ((int64_t(page) * H + h) * G + sub * kTile + 2 * lc) * D + 4 * kVW * lr;
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
          for (int vh = 0; vh < kVH; ++vh)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const uint8_t* at_ = p + (mt * 16 + (t / 2) * 8 + t % 2) * D + 128 * vh;
              const bool there = kWhole || 128 * vh + 4 * kVW * lr < D;
              if constexpr (kVW == 4) {
                const uint4 u = there ? ld_stream(at_) : make_uint4(0, 0, 0, 0);
                vr[mt][vh][t][0] = u.x; vr[mt][vh][t][1] = u.y; vr[mt][vh][t][2] = u.z; vr[mt][vh][t][3] = u.w;
              } else {
                const uint2 u = there ? ld_stream2(at_) : make_uint2(0, 0);
                vr[mt][vh][t][0] = u.x; vr[mt][vh][t][1] = u.y;
              }
            }
        vs = __ldg(c.value_scale + int64_t(page) * H + h);
      };

      bool ok;
      int page = page_at(t0 / per_block, ok);
      load_keys(page, t0 % per_block);
      load_values(page, t0 % per_block);
      for (int t = t0; t < p1; ++t) {
        float s[kNT][kMT][4];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int mt = 0; mt < kMT; ++mt) s[nt][mt][0] = s[nt][mt][1] = s[nt][mt][2] = s[nt][mt][3] = 0.f;
#pragma unroll
        for (int jj = 0; jj < kKC; ++jj)
#pragma unroll
          for (int mt = 0; mt < kMT; ++mt) {
            const uint32_t w0[4] = {kr[mt][0][jj].x, kr[mt][0][jj].y, kr[mt][0][jj].z, kr[mt][0][jj].w};
            const uint32_t w1[4] = {kr[mt][1][jj].x, kr[mt][1][jj].y, kr[mt][1][jj].z, kr[mt][1][jj].w};
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
        const bool more = t + 1 < p1;
        const int sub = (t + 1) % per_block;
        if (more) {
          if (sub == 0) page = page_at((t + 1) / per_block, ok);
          load_keys(page, sub);
        }
        uint32_t wb[kNT][kMT][kParts][2];           // weights as the other operand: tokens 0..7 and 8..15 of a group
        float alpha[kNT][2];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
          for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][mt][i] = ok_now ? s[nt][mt][i] * (fac[nt][i & 1] * ks_now) : -INFINITY;
          softmax(s[nt], nt, alpha[nt]);
          float sum[2] = {0.f, 0.f};
#pragma unroll
          for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint32_t hi = dev::from_f2<false>(s[nt][mt][2 * r], s[nt][mt][2 * r + 1]);
              const float2 back = dev::to_f2<false>(hi);
              wb[nt][mt][0][r] = transpose8x8(hi);
              if constexpr (kParts == 2) {
                wb[nt][mt][kParts - 1][r] =
                    transpose8x8(dev::from_f2<false>(s[nt][mt][2 * r] - back.x, s[nt][mt][2 * r + 1] - back.y));
                sum[0] += s[nt][mt][2 * r];
                sum[1] += s[nt][mt][2 * r + 1];
              } else {                              // the sum of what the product uses
                sum[0] += back.x;
                sum[1] += back.y;
              }
            }
          l[nt][0] = l[nt][0] * alpha[nt][0] + sum[0];
          l[nt][1] = l[nt][1] * alpha[nt][1] + sum[1];
        }
        const float vmul = ok_now ? vs_now : 0.f;
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
                uint32_t a0, a1, a2, a3;
                codes_to_half<kCode>(prmt(vr[mt][vh][0][x], vr[mt][vh][1][x], sel), a0, a1);
                codes_to_half<kCode>(prmt(vr[mt][vh][2][x], vr[mt][vh][3][x], sel), a2, a3);
#pragma unroll
                for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                  for (int p = 0; p < kParts; ++p)
                    mma<false>(acc[nt], a0, a1, a2, a3, wb[nt][mt][p][0], wb[nt][mt][p][1]);
              }
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][i][e] = fmaf(acc[nt][e], vmul, o[nt][i][e] * alpha[nt][e & 1]);
            }
        if (more) load_values(page, sub);
      }
    }

    // ------------------------------------------------------------------ tail: 16 tokens of 16 bits a tile
    if (t1 > tl.paged) {
      if constexpr (kBf16) {                        // q as it is: bf16 products
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
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
      }
      const int64_t base = (int64_t(slot) * H + h) * G * D;
      const uint16_t* tk = static_cast<const uint16_t*>(c.tail_k) + base;
      const uint16_t* tv = static_cast<const uint16_t*>(c.tail_v) + base;
      const float fac16 = a.sm_scale * kLog2e;
      for (int t = max(t0, tl.paged); t < t1; ++t) {
        const int tok = (t - tl.paged) * 16;
        float s[kNT][1][4];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) s[nt][0][0] = s[nt][0][1] = s[nt][0][2] = s[nt][0][3] = 0.f;
        const bool row0 = tok + lr < tl.tail, row1 = tok + lr + 8 < tl.tail;
#pragma unroll
        for (int jj = 0; jj < kKC; ++jj) {
          const uint4 z = make_uint4(0, 0, 0, 0);
          uint4 u[2][2] = {{z, z}, {z, z}};
          const int ch = 64 * jj + 16 * lc;
          if (kWhole || ch < D) {
            const uint16_t* p = tk + (tok + lr) * D + ch;
            if (row0) { u[0][0] = ld_stream(p); u[0][1] = ld_stream(p + 8); }
            if (row1) { u[1][0] = ld_stream(p + 8 * D); u[1][1] = ld_stream(p + 8 * D + 8); }
          }
          const uint32_t w0[8] = {u[0][0].x, u[0][0].y, u[0][0].z, u[0][0].w, u[0][1].x, u[0][1].y, u[0][1].z, u[0][1].w};
          const uint32_t w1[8] = {u[1][0].x, u[1][0].y, u[1][0].z, u[1][0].w, u[1][1].x, u[1][1].y, u[1][1].z, u[1][1].w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
              mma<kBf16>(s[nt][0], w0[2 * i], w1[2 * i], w0[2 * i + 1], w1[2 * i + 1], qf[nt][4 * jj + i][0],
                         qf[nt][4 * jj + i][1]);
        }
        uint32_t wb[kNT][2][2];                     // two parts of the tails' type
        float alpha[kNT][2];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[nt][0][i] = (i < 2 ? row0 : row1) ? s[nt][0][i] * fac16 : -INFINITY;
          softmax(s[nt], nt, alpha[nt]);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t hi = dev::from_f2<kBf16>(s[nt][0][2 * r], s[nt][0][2 * r + 1]);
            const float2 back = dev::to_f2<kBf16>(hi);
            wb[nt][0][r] = transpose8x8(hi);
            wb[nt][1][r] = transpose8x8(dev::from_f2<kBf16>(s[nt][0][2 * r] - back.x, s[nt][0][2 * r + 1] - back.y));
          }
          l[nt][0] = l[nt][0] * alpha[nt][0] + (s[nt][0][0] + s[nt][0][2]);
          l[nt][1] = l[nt][1] * alpha[nt][1] + (s[nt][0][1] + s[nt][0][3]);
        }
#pragma unroll
        for (int vh = 0; vh < kVH; ++vh) {
          // rows behind the tail's end may hold anything: they read as zero
          uint32_t w[4][2 * kVW];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = tok + 2 * lc + (k / 2) * 8 + k % 2;
            const bool there = row < tl.tail && (kWhole || 128 * vh + 4 * kVW * lr < D);
            const uint16_t* p = tv + row * D + 128 * vh + 4 * kVW * lr;
#pragma unroll
            for (int q = 0; q < kVW / 2; ++q) {
              const uint4 u = there ? ld_stream(p + 8 * q) : make_uint4(0, 0, 0, 0);
              w[k][4 * q] = u.x; w[k][4 * q + 1] = u.y; w[k][4 * q + 2] = u.z; w[k][4 * q + 3] = u.w;
            }
          }
#pragma unroll
          for (int x = 0; x < 2 * kVW; ++x) {       // a word holds the channel pair of one output tile
            const int i = vh * kVW * 2 + x;
            const uint32_t a0 = prmt(w[0][x], w[1][x], 0x5410), a1 = prmt(w[0][x], w[1][x], 0x7632);
            const uint32_t a2 = prmt(w[2][x], w[3][x], 0x5410), a3 = prmt(w[2][x], w[3][x], 0x7632);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][i][e] *= alpha[nt][e & 1];
              mma<kBf16>(o[nt][i], a0, a1, a2, a3, wb[nt][0][0], wb[nt][0][1]);
              mma<kBf16>(o[nt][i], a0, a1, a2, a3, wb[nt][1][0], wb[nt][1][1]);
            }
          }
        }
      }
    }

    // ------------------------------------------------------------------ store
    const bool all_here = t0 == 0 && t1 == tl.all;
    const int64_t place = 2 * int64_t(warp) + (f > warp * per_warp);   // the slice's first segment, or its last
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[nt][j];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int qh = nt * 8 + 2 * lc + j;
        if (qh >= heads) continue;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint16_t* out = static_cast<uint16_t*>(a.out) + b * a.out_s_seq + (h * g + q0 + qh) * a.out_s_head;
        float* part = plan.part_o + (place * plan.pass_heads + qh) * D;
        if (!all_here && lr == 0) {
          float* ml = plan.part_ml + (place * plan.pass_heads + qh) * 2;
          ml[0] = m[nt][j];
          ml[1] = sum;
        }
#pragma unroll
        for (int x = 0; x < kOT / 2; ++x) {         // four channels from two output tiles
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
    f = begin + t1;
    if (f == seg_end) {
      begin = seg_end;
      if (++seg == per_row) { seg = 0; ++b; }
    }
  }
}

// One CTA per segment: joins the parts that its warps left, out = sum_i 2^(m_i - M) O_i /
// sum_i 2^(m_i - M) l_i; zeros for an empty slot.  The threads form groups of D / 4 (one
// 16-byte vector of a part each); the groups share the parts and are summed in order.
template <int kTile, bool kBf16>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(KittyKv8AttentionArgs a, Plan plan) {
  extern __shared__ float4 s_sum[];                 // [groups][heads * D / 4]
  __shared__ float s_l[kMergeThreads];
  const KittyKv8Cache& c = a.cache;
  const int D = c.head_dim, g = a.num_q_heads / c.num_heads, per_row = c.num_heads * plan.passes;
  const int b = blockIdx.x / per_row, seg = blockIdx.x % per_row;
  const int h = seg / plan.passes, q0 = (seg % plan.passes) * plan.pass_heads;
  const int heads = min(plan.pass_heads, g - q0);
  // where the segment lies among all tiles
  int64_t before = 0, total = 0;
  {
    const int lane = threadIdx.x & 31;
    for (int i = lane; i < a.batch; i += 32) {
      const int64_t n = tiles_of<kTile>(c, tokens_of(a, i)).all;
      total += n;
      if (i < b) before += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    total *= per_row;
    before *= per_row;
  }
  const int tiles = tiles_of<kTile>(c, tokens_of(a, b)).all;
  uint16_t* out = static_cast<uint16_t*>(a.out) + b * a.out_s_seq + int64_t(h * g + q0) * a.out_s_head;
  const int vecs = D / 4;
  if (tiles == 0) {
    for (int u = threadIdx.x; u < heads * vecs; u += kMergeThreads)
      *reinterpret_cast<uint2*>(out + (u / vecs) * a.out_s_head + (u % vecs) * 4) = make_uint2(0, 0);
    return;
  }
  const int64_t per_warp = (total + plan.warps - 1) / plan.warps;
  const int64_t begin = before + int64_t(seg) * tiles, end = begin + tiles;
  const int w0 = int(begin / per_warp), w1 = int((end - 1) / per_warp);
  if (w0 == w1) return;                             // stored by its warp
  const bool inside = begin > w0 * per_warp;        // it is the last of w0's slice, not the first
  auto place = [&](int w) { return 2 * int64_t(w) + (w == w0 && inside); };
  const int units = heads * vecs;
  const int groups = max(1, kMergeThreads / units);
  for (int u0 = 0; u0 < units; u0 += kMergeThreads) {
    const int group = units <= kMergeThreads ? threadIdx.x / units : 0;
    const int u = u0 + (units <= kMergeThreads ? threadIdx.x % units : threadIdx.x);
    const bool work = u < units && group < groups;
    const int qh = work ? u / vecs : 0, v = u % vecs;
    float top = -INFINITY;
    for (int w = w0; w <= w1; ++w) top = fmaxf(top, plan.part_ml[(place(w) * plan.pass_heads + qh) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    if (work) {
#pragma unroll 4
      for (int w = w0 + group; w <= w1; w += groups) {
        const int64_t at = place(w) * plan.pass_heads + qh;
        const float k = ex2(plan.part_ml[at * 2] - ref);
        const float4 p = *reinterpret_cast<const float4*>(plan.part_o + at * D + v * 4);
        sum = fmaf(k, plan.part_ml[at * 2 + 1], sum);
        acc.x = fmaf(k, p.x, acc.x);
        acc.y = fmaf(k, p.y, acc.y);
        acc.z = fmaf(k, p.z, acc.z);
        acc.w = fmaf(k, p.w, acc.w);
      }
    }
    if (groups > 1) {
      s_sum[threadIdx.x] = acc;
      s_l[threadIdx.x] = sum;
      __syncthreads();
      if (work && group == 0)
        for (int k = 1; k < groups; ++k) {
          const float4 p = s_sum[k * units + u];
          acc.x += p.x; acc.y += p.y; acc.z += p.z; acc.w += p.w;
          sum += s_l[k * units + u];
        }
    }
    if (work && group == 0) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint2*>(out + qh * a.out_s_head + v * 4) =
          make_uint2(dev::from_f2<kBf16>(acc.x * inv, acc.y * inv), dev::from_f2<kBf16>(acc.z * inv, acc.w * inv));
    }
  }
}

// Resident CTAs per SM that a kernel's registers allow (asked once per kernel).
template <int kDim, int kNT, bool kWhole, bool kBf16, int kCode>
int resident() {
  static int known = 0;
  if (known == 0) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attention_kernel<kDim, kNT, kWhole, kBf16, kCode>,
                                                      kWarps * 32, 0) != cudaSuccess || n < 1) {
      cudaGetLastError();
      return 1;
    }
    known = n;
  }
  return known;
}

template <int kDim, int kNT, bool kWhole, bool kBf16, int kCode>
int launch(const KittyKv8AttentionArgs& a, Plan plan, uint32_t* err, cudaStream_t s, int* warps) {
  const int grid = sm_count() * resident<kDim, kNT, kWhole, kBf16, kCode>();
  plan.warps = grid * kWarps;
  if (warps) { *warps = plan.warps; return KITTY_OK; }
  const size_t parts = size_t(2) * plan.warps * plan.pass_heads;
  const size_t ml = (parts * 2 * 4 + 255) / 256 * 256;
  if (a.workspace_bytes < ml + parts * a.cache.head_dim * 4)
    return fail(KITTY_ERR_WORKSPACE, "kv8_attention", "workspace smaller than kitty_kv8_attention_workspace_size()");
  plan.part_ml = static_cast<float*>(a.workspace);
  plan.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + ml);
  attention_kernel<kDim, kNT, kWhole, kBf16, kCode><<<grid, kWarps * 32, 0, s>>>(a, plan, err);
  const int rc = check_launch("kv8_attention");
  if (rc != KITTY_OK) return rc;
  constexpr int kTile = kDim == 256 ? 16 : 32;
  const unsigned segments = unsigned(a.batch) * a.cache.num_heads * plan.passes;
  merge_kernel<kTile, kBf16><<<segments, kMergeThreads, kMergeThreads * sizeof(float4), s>>>(a, plan);
  return check_launch("kv8_attention (merge)");
}

template <int kDim, bool kWhole, bool kBf16, int kCode>
int launch_heads(const KittyKv8AttentionArgs& a, uint32_t* err, cudaStream_t s, int* warps, int* pass_heads) {
  // Query heads of a KV head in passes of 8 or 16: 16 columns share every conversion of
  // a code, but at 256 channels their outputs would not fit the registers.
  const int g = a.num_q_heads / a.cache.num_heads;
  constexpr bool kTwo = kDim <= 128;
  Plan plan{};
  const int most = kTwo && g > 8 ? 16 : 8;
  plan.passes = (g + most - 1) / most;
  plan.pass_heads = (g + plan.passes - 1) / plan.passes;
  if (pass_heads) *pass_heads = plan.pass_heads;
  if constexpr (kTwo) {
    if (plan.pass_heads > 8) return launch<kDim, 2, kWhole, kBf16, kCode>(a, plan, err, s, warps);
  }
  return launch<kDim, 1, kWhole, kBf16, kCode>(a, plan, err, s, warps);
}

template <bool kBf16, int kCode>
int launch_dim(const KittyKv8AttentionArgs& a, uint32_t* err, cudaStream_t s, int* warps, int* ph) {
  const int D = a.cache.head_dim;
  if (D == 64) return launch_heads<64, true, kBf16, kCode>(a, err, s, warps, ph);
  if (D < 64) return launch_heads<64, false, kBf16, kCode>(a, err, s, warps, ph);
  if (D == 128) return launch_heads<128, true, kBf16, kCode>(a, err, s, warps, ph);
  if (D < 128) return launch_heads<128, false, kBf16, kCode>(a, err, s, warps, ph);
  if (D == 256) return launch_heads<256, true, kBf16, kCode>(a, err, s, warps, ph);
  return launch_heads<256, false, kBf16, kCode>(a, err, s, warps, ph);
}

int dispatch(const KittyKv8AttentionArgs& a, uint32_t* err, cudaStream_t s, int* warps, int* ph) {
  if (a.cache.dtype == KITTY_KV8_BF16)
    return a.cache.code == KITTY_KV8_E4M3 ? launch_dim<true, KITTY_KV8_E4M3>(a, err, s, warps, ph)
                                          : launch_dim<true, KITTY_KV8_INT8>(a, err, s, warps, ph);
  return a.cache.code == KITTY_KV8_E4M3 ? launch_dim<false, KITTY_KV8_E4M3>(a, err, s, warps, ph)
                                        : launch_dim<false, KITTY_KV8_INT8>(a, err, s, warps, ph);
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
  if (int64_t(a->batch) * a->num_q_heads > 0x7fffffffLL)
    return fail(KITTY_ERR_UNSUPPORTED, what, "batch * num_q_heads must fit 31 bits");
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
  int warps = 0, ph = 0;
  dispatch(*a, nullptr, nullptr, &warps, &ph);
  const size_t parts = size_t(2) * warps * ph;
  *bytes = (parts * 2 * 4 + 255) / 256 * 256 + parts * a->cache.head_dim * 4;
  return KITTY_OK;
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
  return dispatch(*a, err, as_stream(stream), nullptr, nullptr);
}
