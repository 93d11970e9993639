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
// registers: 2 bytes read and 1 written a value, the floor of this operation.
#include "kv8_common.cuh"

namespace kitty8 {
namespace {

constexpr int kHeld = 4;        // 16-byte vectors a thread holds in registers for each of key and value

// Source rows of a block: the first `have` from the tail, the others from the call's rows.
struct Rows {
  const uint16_t* tail;         // [G][D]
  const uint16_t* fresh;        // row `have` of the block
  int64_t s_row;
  int have;
};

__device__ __forceinline__ uint4 load_vec(const Rows& r, int D, int t, int c) {
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

// Quantise one block of keys and one of values by the whole CTA.
template <bool kBf16, int kCode, int kThreads>
__device__ __forceinline__ void quantise_block(const Rows (&src)[2], uint8_t* const (&codes)[2], float* const (&scale)[2], int G, int D,
                               uint32_t (*s_top)[kThreads / 32]) {
  constexpr float kQ = kCode == KITTY_KV8_E4M3 ? 448.f : 127.f;
  const int tid = threadIdx.x, per = D / 8, vecs = G * per;
  uint4 held[2][kHeld];
  uint32_t top[2] = {0u, 0u};
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int v = tid + i * kThreads;
      held[x][i] = v < vecs ? load_vec(src[x], D, v / per, v % per) : make_uint4(0, 0, 0, 0);
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) top[x] = top_of<kBf16>(held[x][i], top[x]);
    for (int v = tid + kHeld * kThreads; v < vecs; v += kThreads)
      top[x] = top_of<kBf16>(load_vec(src[x], D, v / per, v % per), top[x]);
    top[x] = dev::max2<kBf16>(top[x], (top[x] >> 16) | (top[x] << 16));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top[x] = dev::max2<kBf16>(top[x], __shfl_xor_sync(0xffffffffu, top[x], o));
    if ((tid & 31) == 0) s_top[x][tid >> 5] = top[x];
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    uint32_t m = s_top[x][0];
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) m = dev::max2<kBf16>(m, s_top[x][i]);
    const float a = dev::to_f2<kBf16>(m).x;
    const float top_f = a < 0x1p-100f ? 0x1p-100f : a;       // NaN stays
    const float r = __frcp_rn(top_f) * kQ;                   // each factor rounded once
    if (tid == 0) *scale[x] = top_f * (1.f / kQ);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int v = tid + i * kThreads;
      if (v < vecs) reinterpret_cast<uint2*>(codes[x])[v] = encode_vec<kBf16, kCode>(held[x][i], r);
    }
    for (int v = tid + kHeld * kThreads; v < vecs; v += kThreads)
      reinterpret_cast<uint2*>(codes[x])[v] = encode_vec<kBf16, kCode>(load_vec(src[x], D, v / per, v % per), r);
  }
}

// Entry i's slot, its rows [o, o + len) and the tokens it has; false (and flagged) if any
// of them is out of range, or the slot is an earlier entry's.
__device__ __forceinline__ bool entry_of(const KittyKv8WriteArgs& a, int i, bool first_cta, uint32_t* err, int& slot,
                                         int& o, int& len, int& cached) {
  uint32_t bad = 0;
  slot = a.seq_map ? a.seq_map[i] : i;
  o = a.row_offsets ? a.row_offsets[i] : i;
  const int64_t given = a.row_offsets ? int64_t(a.row_offsets[i + 1]) - o : 1;
  len = int(given);
  if (slot < 0 || slot >= a.cache.slots) {
    bad = kErrSlot;
  } else {
    if (a.seq_map && dev::repeated(a.seq_map, i, slot)) bad = kErrSlot;
    cached = a.cache.lengths[slot];
    if (cached < 0 || cached > 0x7fffffff - a.rows) bad |= kErrLength;
  }
  if (o < 0 || given < 0 || o + given > a.rows) bad |= kErrRows;
  if (bad && first_cta && threadIdx.x == 0) dev::flag(err, bad);
  return bad == 0;
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

template <bool kBf16, int kCode, int kThreads>
__global__ void __launch_bounds__(kThreads) write_kernel(KittyKv8WriteArgs a, uint32_t* err) {
  __shared__ uint32_t s_top[2][kThreads / 32];
  const KittyKv8Cache& c = a.cache;
  const int G = c.page_size, D = c.head_dim, h = blockIdx.y;
  const int64_t block_elems = int64_t(G) * D;
  int slot, o, len, cached;
  int block, have, skip;        // the block to quantise: its tail rows, and the entry's rows before its first new row
  bool whole;
  const bool entry_cta = int(blockIdx.x) < a.n;
  if (entry_cta) {
    if (!entry_of(a, blockIdx.x, h == 0, err, slot, o, len, cached)) return;
    block = cached / G;
    have = cached % G;
    skip = 0;
    whole = have > 0 && have + len >= G;
  } else {
    const int64_t last = int64_t(int(blockIdx.x) - a.n) * G + G - 1;   // < rows by the grid's size
    const int i = dev::count_le(a.row_offsets, a.n + 1, int(last)) - 1;
    if (i < 0 || i >= a.n) return;                                     // rows behind the last entry
    if (!entry_of(a, i, false, err, slot, o, len, cached)) return;
    const int64_t local = last - o;
    if (local < 0 || local >= len) return;
    block = int((cached + local) / G);
    have = 0;
    const int64_t first = int64_t(block) * G - cached;
    whole = first >= 0 && first + G <= len;
    if (!whole) return;
    skip = int(first);
  }
  const int64_t tail = (int64_t(slot) * c.num_heads + h) * block_elems;
  uint16_t* tails[2] = {static_cast<uint16_t*>(c.tail_k) + tail, static_cast<uint16_t*>(c.tail_v) + tail};
  const int64_t s_row[2] = {a.k_s_row, a.v_s_row};
  const uint16_t* rows[2] = {static_cast<const uint16_t*>(a.key) + int64_t(o) * a.k_s_row + h * a.k_s_head,
                             static_cast<const uint16_t*>(a.value) + int64_t(o) * a.v_s_row + h * a.v_s_head};
  if (whole) {
    const int page = page_of(c, slot, block, err);
    if (page >= 0) {
      const int64_t at = int64_t(page) * c.num_heads + h;
      const Rows src[2] = {{tails[0], rows[0] + skip * s_row[0], s_row[0], have},
                           {tails[1], rows[1] + skip * s_row[1], s_row[1], have}};
      uint8_t* const codes[2] = {static_cast<uint8_t*>(c.key_codes) + at * block_elems,
                                 static_cast<uint8_t*>(c.value_codes) + at * block_elems};
      float* const scale[2] = {c.key_scale + at, c.value_scale + at};
      quantise_block<kBf16, kCode, kThreads>(src, codes, scale, G, D, s_top);
    }
  }
  if (!entry_cta) return;
  // the rows that fill no block: behind the tail's, or from its first row if a block was completed
  const int left = have + len < G ? len : int((int64_t(cached) + len) % G);
  const int to = have + len < G ? have : 0;
  if (left == 0) return;
  if (whole) __syncthreads();   // every thread has read the tail rows of the block
  const int per = D / 8;
  for (int u = threadIdx.x; u < 2 * left * per; u += kThreads) {
    const int x = u >= left * per, v = u - x * left * per, t = v / per, d = v % per;
    const uint16_t* src = x ? rows[1] + int64_t(len - left + t) * s_row[1] : rows[0] + int64_t(len - left + t) * s_row[0];
    reinterpret_cast<uint4*>((x ? tails[1] : tails[0]) + (to + t) * D)[d] = reinterpret_cast<const uint4*>(src)[d];
  }
}

template <bool kBf16, int kCode>
int launch(const KittyKv8WriteArgs& a, uint32_t* err, cudaStream_t s) {
  const int64_t windows = a.row_offsets ? a.rows / a.cache.page_size : 0;
  const dim3 grid(unsigned(a.n + windows), unsigned(a.cache.num_heads));
  if (windows) write_kernel<kBf16, kCode, 256><<<grid, 256, 0, s>>>(a, err);
  else write_kernel<kBf16, kCode, 128><<<grid, 128, 0, s>>>(a, err);   // mostly single rows: 2 D / 8 threads copy
  return check_launch("kv8_write");
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
    return a->cache.code == KITTY_KV8_E4M3 ? launch<true, KITTY_KV8_E4M3>(*a, err, s)
                                           : launch<true, KITTY_KV8_INT8>(*a, err, s);
  return a->cache.code == KITTY_KV8_E4M3 ? launch<false, KITTY_KV8_E4M3>(*a, err, s)
                                         : launch<false, KITTY_KV8_INT8>(*a, err, s);
}
