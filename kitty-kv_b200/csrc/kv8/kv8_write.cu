// Quantising the cache as it is written: new key / value rows go to the tails, and the
// blocks of G tokens that they fill to 8-bit pages, in one launch without a plan.
//
// Who quantises what follows from the row offsets alone.  CTA x < n belongs to entry x:
// it completes the block that its slot had begun (tail rows and new rows together) and
// then stores the rows that fill no block in the tail; one CTA does both, because the
// second may overwrite rows that the first reads.  CTA n + w looks at the w-th window of
// G rows: a block that lies in the new rows as a whole contains exactly one row whose
// index is G - 1 modulo G, so the block with the window's last row, if it is whole, is
// that CTA's, and each is found once.
//
// A block of one head (G x D values) is read once into registers where it fits, its
// largest magnitude taken with packed 16-bit maxima (exact), and the codes stored from
// registers: 2 bytes read and 1 written a value, the floor of this operation.  (With one head a
// CTA, where each place of a block stands three times in the code, 64 registers do not hold all
// of it: 88 bytes a thread are spilled.)  Of small blocks a CTA takes several heads, so that its
// threads have as much to do.
#include "kv8_common.cuh"

namespace kitty8 {
namespace {

constexpr int kHeld = 4;        // 16-byte vectors a thread holds in registers for each of key and value
constexpr int kThreads = 256;
constexpr int kMinCtas = 4;     // resident on an SM: 75K ragged rows take 108 us at 2, 86 at 3, 76 at 4, 95 at 5
constexpr int kStepEntries = 8; // entries of a decode step whose blocks one CTA looks after

// Source rows of a block: the first `have` from the tail, the others from the call's rows.
struct Rows {
  const uint16_t* tail;         // [G][D]
  const uint16_t* fresh;        // row `have` of the block
  int64_t s_row;
  int have;
};

// 16-byte vectors of a row: known when compiled for the usual head sizes, so that finding
// a vector's row takes a shift and not a division.
template <int kPer>
__device__ __forceinline__ int vecs_of_row(int D) { return kPer ? kPer : D / 8; }

template <int kPer>
__device__ __forceinline__ uint4 load_vec(const Rows& r, int D, int v) {
  const int per = vecs_of_row<kPer>(D), t = v / per, c = v - t * per;
  const uint16_t* p = t < r.have ? r.tail + t * D : r.fresh + int64_t(t - r.have) * r.s_row;
  return *(reinterpret_cast<const uint4*>(p) + c);
}

template <bool kBf16>
__device__ __forceinline__ uint32_t top_of(const uint4& v, uint32_t top) {
  top = dev::max2<kBf16>(top, dev::abs2(v.x));
  top = dev::max2<kBf16>(top, dev::abs2(v.y));
  top = dev::max2<kBf16>(top, dev::abs2(v.z));
  return dev::max2<kBf16>(top, dev::abs2(v.w));
}

template <bool kBf16, int kCode>
__device__ __forceinline__ uint2 encode_vec(const uint4& v, float r) {
  const float2 a = dev::to_f2<kBf16>(v.x), b = dev::to_f2<kBf16>(v.y), c = dev::to_f2<kBf16>(v.z),
               d = dev::to_f2<kBf16>(v.w);
  return make_uint2(dev::encode4<kCode>(a.x * r, a.y * r, b.x * r, b.y * r),
                    dev::encode4<kCode>(c.x * r, c.y * r, d.x * r, d.y * r));
}

// The page of block b of a slot; -1 (and flagged) if the cache has none.
__device__ __forceinline__ int page_of(const KittyKv8Cache& c, int slot, int b, uint32_t* err) {
  int page = -1;
  if (b < c.max_pages) page = c.block_table[int64_t(slot) * c.bt_s_slot + b];
  if (page < 0 || page >= c.pages) {
    if (threadIdx.x == 0) dev::flag(err, kErrPage);
    return -1;
  }
  return page;
}

// Quantise block `block` of a slot's head h from kX kinds of rows (keys, values, or both at
// once) by the whole CTA.  The rows are asked for first and the page looked up while they are
// on their way.
template <bool kBf16, int kCode, int kPer, int kX>
__device__ __forceinline__ void quantise_rows(const KittyKv8Cache& c, int slot, int block, int h, const Rows* src,
                                              void* const* pools, float* const* scales, uint32_t (*s_top)[kThreads / 32],
                                              uint32_t* err) {
  constexpr float kQ = kCode == KITTY_KV8_E4M3 ? 448.f : 127.f;
  const int G = c.page_size, D = c.head_dim, tid = threadIdx.x, vecs = G * vecs_of_row<kPer>(D);
  uint4 held[kX][kHeld];
  uint32_t top[kX];
#pragma unroll
  for (int x = 0; x < kX; ++x) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int v = tid + i * kThreads;
      held[x][i] = v < vecs ? load_vec<kPer>(src[x], D, v) : make_uint4(0, 0, 0, 0);
    }
  }
  const int page = page_of(c, slot, block, err);
  if (page < 0) return;
#pragma unroll
  for (int x = 0; x < kX; ++x) {
    top[x] = 0u;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) top[x] = top_of<kBf16>(held[x][i], top[x]);
    for (int v = tid + kHeld * kThreads; v < vecs; v += kThreads) top[x] = top_of<kBf16>(load_vec<kPer>(src[x], D, v), top[x]);
    top[x] = dev::max2<kBf16>(top[x], (top[x] >> 16) | (top[x] << 16));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top[x] = dev::max2<kBf16>(top[x], __shfl_xor_sync(0xffffffffu, top[x], o));
    if ((tid & 31) == 0) s_top[x][tid >> 5] = top[x];
  }
  __syncthreads();
  const int64_t at = int64_t(page) * c.num_heads + h;
#pragma unroll
  for (int x = 0; x < kX; ++x) {
    uint32_t m = s_top[x][0];
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) m = dev::max2<kBf16>(m, s_top[x][i]);
    const float a = dev::to_f2<kBf16>(m).x;
    const float top_f = a < 0x1p-100f ? 0x1p-100f : a;       // NaN stays
    const float r = __frcp_rn(top_f) * kQ;                   // each factor rounded once
    if (tid == 0) scales[x][at] = top_f * (1.f / kQ);
    uint2* codes = reinterpret_cast<uint2*>(static_cast<uint8_t*>(pools[x]) + at * G * D);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int v = tid + i * kThreads;
      if (v < vecs) codes[v] = encode_vec<kBf16, kCode>(held[x][i], r);
    }
    for (int v = tid + kHeld * kThreads; v < vecs; v += kThreads)
      codes[v] = encode_vec<kBf16, kCode>(load_vec<kPer>(src[x], D, v), r);
  }
}

// Keys and values together where they fit the registers.  A larger block is read twice, the
// second time from L2, and one kind after the other keeps what is in use small enough for it
// (29K tokens, 4 heads of 256, 256-token pages: 46 us, both kinds together 63; 8 of 128: 40 and
// 44; 75K tokens of 8 of 128 in 128-token pages: 86 and 84).
template <bool kBf16, int kCode, int kPer>
__device__ __forceinline__ void quantise_block(const KittyKv8Cache& c, int slot, int block, int h, const Rows (&src)[2],
                                               uint32_t (*s_top)[kThreads / 32], uint32_t* err) {
  void* const pools[2] = {c.key_codes, c.value_codes};
  float* const scales[2] = {c.key_scale, c.value_scale};
  if (c.page_size * vecs_of_row<kPer>(c.head_dim) <= kHeld * kThreads) {
    quantise_rows<kBf16, kCode, kPer, 2>(c, slot, block, h, src, pools, scales, s_top, err);
  } else {
    quantise_rows<kBf16, kCode, kPer, 1>(c, slot, block, h, src, pools, scales, s_top, err);
    __syncthreads();
    quantise_rows<kBf16, kCode, kPer, 1>(c, slot, block, h, src + 1, pools + 1, scales + 1, s_top, err);
  }
}

// The same for a block's heads h .. h + heads - 1 (at most 2^shift), 2^-shift of the CTA's warps
// for each, whose registers hold it.  kShift: the shift, known when compiled (75K ragged rows of
// 8 heads of 128 in 32-token pages: 74 us, 84 otherwise), or -1.
template <bool kBf16, int kCode, int kPer, int kShift>
__device__ __forceinline__ void quantise_heads(const KittyKv8Cache& c, int slot, int block, int h, int heads, int shift_,
                                               const Rows (&src)[2], const int64_t (&s_head)[2],
                                               uint32_t (*s_top)[kThreads / 32], uint32_t* err) {
  constexpr float kQ = kCode == KITTY_KV8_E4M3 ? 448.f : 127.f;
  const int G = c.page_size, D = c.head_dim, vecs = G * vecs_of_row<kPer>(D);
  const int shift = kShift < 0 ? shift_ : kShift, threads = kThreads >> shift, hh = threadIdx.x / threads, tid = threadIdx.x - hh * threads;
  uint4 held[2][kHeld];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const Rows r{src[x].tail + int64_t(hh) * G * D, src[x].fresh + hh * s_head[x], src[x].s_row, src[x].have};
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int v = tid + i * threads;
      held[x][i] = hh < heads && v < vecs ? load_vec<kPer>(r, D, v) : make_uint4(0, 0, 0, 0);
    }
  }
  const int page = page_of(c, slot, block, err);
  if (page < 0) return;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) top = top_of<kBf16>(held[x][i], top);
    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));     // (as integers NaN is above infinity)
    if ((threadIdx.x & 31) == 0) s_top[x][threadIdx.x >> 5] = top;
  }
  __syncthreads();
  if (hh >= heads) return;
  const int64_t at = int64_t(page) * c.num_heads + h + hh;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < threads / 32; ++i) m = max(m, s_top[x][hh * (threads / 32) + i]);
    const float a = dev::to_f2<kBf16>(m).x;
    const float top_f = a < 0x1p-100f ? 0x1p-100f : a;
    const float r = __frcp_rn(top_f) * kQ;
    if (tid == 0) (x ? c.value_scale : c.key_scale)[at] = top_f * (1.f / kQ);
    uint2* codes = reinterpret_cast<uint2*>(static_cast<uint8_t*>(x ? c.value_codes : c.key_codes) + at * G * D);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int v = tid + i * threads;
      if (v < vecs) codes[v] = encode_vec<kBf16, kCode>(held[x][i], r);
    }
  }
}

// Entry i's slot, its rows [o, o + len) and the tokens it has; false for padding (a negative
// slot), and (flagged) if any of them is out of range, or the slot is an earlier entry's.  The
// offsets of padding are looked at too: rows are searched for among those of all entries.
__device__ __forceinline__ bool entry_of(const KittyKv8WriteArgs& a, int i, bool first_cta, uint32_t* err, int& slot,
                                         int& o, int& len, int& cached) {
  uint32_t bad = 0;
  slot = a.seq_map ? a.seq_map[i] : i;
  if (slot < 0 && !a.row_offsets) return false;
  o = a.row_offsets ? a.row_offsets[i] : i;
  const int64_t given = a.row_offsets ? int64_t(a.row_offsets[i + 1]) - o : 1;
  len = int(given);
  if (slot >= a.cache.slots) {
    bad = kErrSlot;
  } else if (slot >= 0) {
    if (a.seq_map && dev::repeated(a.seq_map, i, slot)) bad = kErrSlot;
    cached = a.cache.lengths[slot];
    if (cached < 0 || cached > 0x7fffffff - a.rows) bad |= kErrLength;
  }
  if (o < 0 || given < 0 || o + given > a.rows) bad |= kErrRows;
  if (bad && first_cta && threadIdx.x == 0) dev::flag(err, bad);
  return bad == 0 && slot >= 0;
}

__device__ __forceinline__ const uint16_t* row_of(const void* base, int64_t row, int64_t s_row, int64_t h, int64_t s_head) {
  return static_cast<const uint16_t*>(base) + row * s_row + h * s_head;
}

// Ragged rows; each CTA 2^kShift heads (-1: 2^shift).  CTAs run over the heads first: those that are resident together read whole
// rows of the tokens, and not one head's slice of many.
template <bool kBf16, int kCode, int kPer, int kShift>
__global__ void __launch_bounds__(kThreads, kMinCtas) write_kernel(KittyKv8WriteArgs a, int shift_, uint32_t* err) {
  __shared__ uint32_t s_top[2][kThreads / 32];
  dev::wait_for_stream();
  const KittyKv8Cache& c = a.cache;
  const int G = c.page_size, D = c.head_dim;
  const int shift = kShift < 0 ? shift_ : kShift, groups = (c.num_heads + (1 << shift) - 1) >> shift;
  const int item = blockIdx.x / groups, h = (blockIdx.x - item * groups) << shift;
  const int heads = min(1 << shift, c.num_heads - h);
  [[maybe_unused]] const int64_t s_head[2] = {a.k_s_head, a.v_s_head};
  int slot, o, len, cached;
  if (item < a.n) {
    if (!entry_of(a, item, h == 0, err, slot, o, len, cached)) return;
    const int block = cached / G, have = cached - block * G;
    const bool whole = have > 0 && have + len >= G;
    // the rows that fill no block: behind the tail's, or from its first row if a block was completed
    const int left = have + len < G ? len : int((int64_t(cached) + len) % G);
    const int to = have + len < G ? have : 0, per = vecs_of_row<kPer>(D);
    const int64_t tail = (int64_t(slot) * c.num_heads + h) * G * D;
    uint16_t* const tail_k = static_cast<uint16_t*>(c.tail_k) + tail;
    uint16_t* const tail_v = static_cast<uint16_t*>(c.tail_v) + tail;
    if (whole) {
      const Rows src[2] = {{tail_k, row_of(a.key, o, a.k_s_row, h, a.k_s_head), a.k_s_row, have},
                           {tail_v, row_of(a.value, o, a.v_s_row, h, a.v_s_head), a.v_s_row, have}};
      if constexpr (kShift != 0)
        quantise_heads<kBf16, kCode, kPer, kShift>(c, slot, block, h, heads, shift, src, s_head, s_top, err);
      else
        quantise_block<kBf16, kCode, kPer>(c, slot, block, h, src, s_top, err);
      __syncthreads();   // every thread has read the tail rows of the block
    }
    for (int hh = 0; hh < heads; ++hh)
      for (int u = threadIdx.x; u < 2 * left * per; u += kThreads) {
        const int x = u >= left * per, v = u - x * left * per, t = v / per, d = v - t * per;
        const uint16_t* src = x ? row_of(a.value, o + len - left + t, a.v_s_row, h + hh, a.v_s_head)
                                : row_of(a.key, o + len - left + t, a.k_s_row, h + hh, a.k_s_head);
        reinterpret_cast<uint4*>((x ? tail_v : tail_k) + (hh * G + to + t) * D)[d] = reinterpret_cast<const uint4*>(src)[d];
      }
  } else {
    const int64_t last = int64_t(item - a.n) * G + G - 1;              // < rows by the grid's size
    const int i = dev::count_le(a.row_offsets, a.n + 1, int(last)) - 1;
    if (i < 0 || i >= a.n) return;                                     // rows behind the last entry
    if (!entry_of(a, i, false, err, slot, o, len, cached)) return;
    const int64_t local = last - o;
    if (local < 0 || local >= len) return;
    const int block = int((cached + local) / G);
    const int64_t first = int64_t(block) * G - cached;                 // the entry's row that the block begins with
    if (first < 0 || first + G > len) return;
    const Rows src[2] = {{nullptr, row_of(a.key, o + first, a.k_s_row, h, a.k_s_head), a.k_s_row, 0},
                         {nullptr, row_of(a.value, o + first, a.v_s_row, h, a.v_s_head), a.v_s_row, 0}};
    if constexpr (kShift != 0)
      quantise_heads<kBf16, kCode, kPer, kShift>(c, slot, block, h, heads, shift, src, s_head, s_top, err);
    else
      quantise_block<kBf16, kCode, kPer>(c, slot, block, h, src, s_top, err);
  }
}

// One row for each entry, a decode step.  The first CTAs look at one head of kStepEntries
// entries and quantise the blocks that this row completes (one in G, when the lengths are
// spread); the others copy an entry's row into the tails, all heads at once.  One CTA for
// each entry and head took 10.4 us for 256 entries and 8 heads: 2048 CTAs, most of which
// copy 512 bytes.
template <bool kBf16, int kCode, int kPer>
__global__ void __launch_bounds__(kThreads, kMinCtas) write_step_kernel(KittyKv8WriteArgs a, uint32_t* err) {
  __shared__ uint32_t s_top[2][kThreads / 32];
  dev::wait_for_stream();
  const KittyKv8Cache& c = a.cache;
  const int G = c.page_size, D = c.head_dim, H = c.num_heads, per = vecs_of_row<kPer>(D);
  const int groups = (a.n + kStepEntries - 1) / kStepEntries;
  int slot, o, len, cached;
  if (int(blockIdx.x) < groups * H) {
    const int group = blockIdx.x / H, h = blockIdx.x - group * H, lane = threadIdx.x & 31;
    // every warp looks at the group's lengths, one a lane
    const int i0 = group * kStepEntries;
    bool full = false;
    if (lane < kStepEntries && i0 + lane < a.n) {
      const int s = a.seq_map ? a.seq_map[i0 + lane] : i0 + lane;
      const int n = s >= 0 && s < c.slots ? c.lengths[s] : -1;
      full = n >= 0 && n % G == G - 1;
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, full); todo; todo &= todo - 1) {
      if (!entry_of(a, i0 + __ffs(todo) - 1, false, err, slot, o, len, cached)) continue;
      const int64_t tail = (int64_t(slot) * H + h) * G * D;
      const Rows src[2] = {{static_cast<const uint16_t*>(c.tail_k) + tail, row_of(a.key, o, a.k_s_row, h, a.k_s_head),
                            a.k_s_row, G - 1},
                           {static_cast<const uint16_t*>(c.tail_v) + tail, row_of(a.value, o, a.v_s_row, h, a.v_s_head),
                            a.v_s_row, G - 1}};
      quantise_block<kBf16, kCode, kPer>(c, slot, cached / G, h, src, s_top, err);
      __syncthreads();   // s_top is used again
    }
    return;
  }
  const int i = blockIdx.x - groups * H, vecs = H * per;
  auto source = [&](int u) {     // vector u of the entry's key row and then its value row
    const int x = u >= vecs, v = u - x * vecs, h = v / per;
    return *(reinterpret_cast<const uint4*>(x ? row_of(a.value, i, a.v_s_row, h, a.v_s_head)
                                              : row_of(a.key, i, a.k_s_row, h, a.k_s_head)) + (v - h * per));
  };
  int u = threadIdx.x;
  uint4 w = u < 2 * vecs ? source(u) : make_uint4(0, 0, 0, 0);     // on its way while the entry is looked up
  if (!entry_of(a, i, true, err, slot, o, len, cached)) return;
  const int row = cached % G;
  if (row == G - 1) return;      // quantised with its block
  for (; u < 2 * vecs; u += kThreads) {
    if (u >= kThreads) w = source(u);
    const int x = u >= vecs, v = u - x * vecs, h = v / per;
    uint16_t* tail = static_cast<uint16_t*>(x ? c.tail_v : c.tail_k) + ((int64_t(slot) * H + h) * G + row) * D;
    reinterpret_cast<uint4*>(tail)[v - h * per] = w;
  }
}

template <bool kBf16, int kCode, int kPer>
int launch(const KittyKv8WriteArgs& a, uint32_t* err, cudaStream_t s) {
  const int64_t H = a.cache.num_heads, items = int64_t(a.n) + a.rows / a.cache.page_size;
  const int64_t steps = (int64_t(a.n) + kStepEntries - 1) / kStepEntries * H + a.n;
  // Heads of a CTA: as many as its registers hold, unless fewer than the card's CTAs are left
  // to share the work.  75K ragged rows of 8 heads of 64 in 32-token pages take 39 us, with one
  // head each 113; 300 rows 3.0, with four heads each 4.0.
  const int vecs = a.cache.page_size * a.cache.head_dim / 8;
  int shift = 0;
  const auto ctas = [&] { return items * ((H + (1 << shift) - 1) >> shift); };
  while (shift < 3 && (vecs << (shift + 1)) <= kHeld * kThreads && (1 << shift) < H &&
         ctas() > int64_t(sm_count()) * kMinCtas)
    ++shift;
  const int64_t grid = a.row_offsets ? ctas() : steps;
  if (grid > 0x7fffffff) return fail(KITTY_ERR_UNSUPPORTED, "kv8_write", "too many rows times heads for one launch");
  const auto go = [&](auto kernel, auto... args) {
    return launch_dependent("kv8_write", kernel, dim3(unsigned(grid)), kThreads, 0, s, a, args..., err);
  };
  if (!a.row_offsets) return go(write_step_kernel<kBf16, kCode, kPer>);
  if (shift == 0) return go(write_kernel<kBf16, kCode, kPer, 0>, 0);
  if constexpr (kPer == 0) return go(write_kernel<kBf16, kCode, 0, -1>, shift);
  if constexpr (kPer == 8)
    if (shift == 2) return go(write_kernel<kBf16, kCode, 8, 2>, 2);
  if constexpr (kPer == 8 || kPer == 16) return go(write_kernel<kBf16, kCode, kPer, 1>, 1);
  return fail(KITTY_ERR_UNSUPPORTED, "kv8_write", "no kernel");     // (the smallest block of 256 channels fills the registers)
}

template <bool kBf16, int kCode>
int launch_dim(const KittyKv8WriteArgs& a, uint32_t* err, cudaStream_t s) {
  if (a.cache.head_dim == 64) return launch<kBf16, kCode, 8>(a, err, s);
  if (a.cache.head_dim == 128) return launch<kBf16, kCode, 16>(a, err, s);
  if (a.cache.head_dim == 256) return launch<kBf16, kCode, 32>(a, err, s);
  return launch<kBf16, kCode, 0>(a, err, s);
}

}  // namespace
}  // namespace kitty8

using namespace kitty8;

extern "C" int kitty_kv8_write(const KittyKv8WriteArgs* a, void* stream) {
  const char* what = "kv8_write";
  if (!a) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "args is NULL");
  const int rc = check_cache(&a->cache, what);
  if (rc != KITTY_OK) return rc;
  if (a->n < 0 || a->rows < 0) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "negative size");
  if (a->n > 0x7fffff00) return fail(KITTY_ERR_UNSUPPORTED, what, "too many entries");     // n + 32 is an int
  if (!a->row_offsets && a->n != a->rows)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "without row_offsets there is one row for each entry");
  if (!a->seq_map && a->n > a->cache.slots)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "more entries than slots");
  if (a->n == 0 || a->rows == 0) return KITTY_OK;
  if (!a->key || !a->value) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "NULL key or value");
  if (!aligned(a->key, 16) || !aligned(a->value, 16) || a->k_s_row % 8 || a->k_s_head % 8 || a->v_s_row % 8 ||
      a->v_s_head % 8)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what,
                "key and value rows must be 16-byte aligned (strides multiples of 8 elements)");
  uint32_t* err = error_word();
  if (!err) return fail(KITTY_ERR_CUDA, what, "no CUDA device");
  cudaStream_t s = as_stream(stream);
  if (a->cache.dtype == KITTY_KV8_BF16)
    return a->cache.code == KITTY_KV8_E4M3 ? launch_dim<true, KITTY_KV8_E4M3>(*a, err, s)
                                           : launch_dim<true, KITTY_KV8_INT8>(*a, err, s);
  return a->cache.code == KITTY_KV8_E4M3 ? launch_dim<false, KITTY_KV8_E4M3>(*a, err, s)
                                         : launch_dim<false, KITTY_KV8_INT8>(*a, err, s);
}
