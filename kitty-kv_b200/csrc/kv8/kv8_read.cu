// Reading the cache back to 16-bit rows.
//
// A CTA takes kRows output rows (tokens, all heads).  Its first warp finds each row's slot
// and page and leaves them in shared memory: 32 entries' offsets, slots and first tokens are
// loaded at once and searched by shuffles, then the row's page and its slot's length, also at
// once.  (A search in memory is a chain of loads, 5 for 24 entries: 24 ragged chunks are
// written and read in 16.4 us so, 16.8 with it; one entry of 4137 tokens in 8.9 and 8.5.  With
// the length first and the page behind it, 16 x 32768 tokens took 576 us instead of 507.)
// Then every thread turns eight codes of keys and of values (8 bytes each) into 16-byte
// stores, contiguous over the row, at the same place of one row after another.  Bound by
// HBM: 1 byte read and 2 written a value.
#include "kv8_common.cuh"

namespace kitty8 {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;      // rows whose loads a thread has in flight

constexpr int64_t kManyValues = 5 * 32 * 1024;   // keys for each SM: five CTAs of 32 rows of 1024

struct RowAt {
  int64_t base;        // element offset of (row, head 0, channel 0) in the pools or the tails
  int32_t page;        // -1: a tail row, -2: nothing to do
};

template <bool kBf16, int kCode, int kRows>
__global__ void __launch_bounds__(kThreads) read_kernel(KittyKv8ReadArgs a, uint32_t* err) {
  __shared__ RowAt s_row[kRows];
  dev::wait_for_stream();
  const KittyKv8Cache& c = a.cache;
  const int G = c.page_size, D = c.head_dim, H = c.num_heads;
  const int64_t r0 = int64_t(blockIdx.x) * kRows;
  const int count = int(min(int64_t(kRows), a.rows - r0));
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, r = int(r0) + min(lane, count - 1);
    const int at0 = a.n < 32 ? 0 : max(dev::count_le(a.row_offsets, a.n + 1, int(r0)) - 1, 0);
    const int e = at0 + lane;            // this lane's entry of the window
    const int offset = e <= a.n ? a.row_offsets[e] : 0x7fffffff;
    const int window_slot = e < a.n && a.seq_map ? a.seq_map[e] : e, window_first = e < a.n && a.first ? a.first[e] : 0;
    int lo = 0;                          // how many of the window's offsets are <= r
#pragma unroll
    for (int step = 16; step > 0; step >>= 1)
      if (__shfl_sync(0xffffffffu, offset, lo + step - 1) <= r) lo += step;
    if (__shfl_sync(0xffffffffu, offset, lo) <= r) ++lo;          // (31 of them, or 32)
    const int from = max(lo - 1, 0);
    int i = at0 + lo - 1, o = __shfl_sync(0xffffffffu, offset, from), slot = __shfl_sync(0xffffffffu, window_slot, from),
        first = __shfl_sync(0xffffffffu, window_first, from), end = __shfl_sync(0xffffffffu, offset, min(from + 1, 31));
    if (from == 31) end = i < a.n ? a.row_offsets[i + 1] : 0;
    if (lo == 32 && at0 + 32 <= a.n) {   // the row is behind the window: many entries of no or few rows
      int hi = a.n + 1;
      lo = at0 + 32;
      while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (a.row_offsets[mid] <= r) lo = mid + 1;
        else hi = mid;
      }
      i = lo - 1;
      o = a.row_offsets[i];
      if (i < a.n) {
        end = a.row_offsets[i + 1];
        slot = a.seq_map ? a.seq_map[i] : i;
        first = a.first ? a.first[i] : 0;
      }
    }
    RowAt at{0, -2};
    uint32_t bad = 0;
    if (i >= 0 && i < a.n) {
      if (o < 0 || o > r || end <= r) {       // (offsets that decrease)
        bad = kErrRows;
      } else if (slot >= c.slots) {
        bad = kErrSlot;
      } else if (slot >= 0) {                 // (a negative slot is padding)
        const int64_t t = int64_t(first) + (r - o);
        const bool fits = t >= 0 && t <= 0x7fffffff;
        const int b = fits ? int(t) / G : 0, in = fits ? int(t) - b * G : 0;
        const int page = fits && b < c.max_pages ? c.block_table[int64_t(slot) * c.bt_s_slot + b] : -1;
        const int len = c.lengths[slot];      // on its way together with the page
        if (!fits || t >= len || len / G > c.max_pages) bad = kErrLength;
        else if (b >= len / G) at = RowAt{(int64_t(slot) * H * G + in) * D, -1};
        else if (page < 0 || page >= c.pages) bad = kErrPage;
        else at = RowAt{(int64_t(page) * H * G + in) * D, page};
      }
    }
    if (lane < count) {
      if (bad) dev::flag(err, bad);
      s_row[lane] = at;
    }
  } else {                               // the other warps look all offsets over
    uint32_t bad = 0;
    for (int64_t i = int64_t(blockIdx.x) * (kThreads - 32) + threadIdx.x - 32; i < a.n; i += int64_t(gridDim.x) * (kThreads - 32)) {
      const int o = a.row_offsets[i], end = a.row_offsets[i + 1];
      if (o < 0 || end < o || end > a.rows) bad = kErrRows;
    }
    if (bad) dev::flag(err, bad);
  }
  __syncthreads();
  const int per = D / 8, vecs = H * per;
  const int64_t s_head = int64_t(G) * D;
  // the threads lie over as many rows as fit, or several times over one
  const int at_once = max(1, kThreads / vecs), row0 = vecs <= kThreads ? threadIdx.x / vecs : 0;
  if (row0 >= at_once) return;
  for (int v = vecs <= kThreads ? threadIdx.x - row0 * vecs : threadIdx.x; v < vecs; v += kThreads) {
    const int h = v / per;
    const int64_t place = h * s_head + (v - h * per) * 8;
    for (int r = row0; r < count; r += at_once * kUnroll) {
      uint2 w[kUnroll][2];
      float sc[kUnroll][2];
      int page[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int row = r + k * at_once;
        page[k] = -2;
        if (row < count) {
          const RowAt at = s_row[row];
          const int64_t off = at.base + place, to = (r0 + row) * vecs + v;
          page[k] = at.page;
          if (at.page >= 0) {
            const int64_t scale = int64_t(at.page) * H + h;
            w[k][0] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(c.key_codes) + off);
            w[k][1] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(c.value_codes) + off);
            sc[k][0] = c.key_scale[scale];
            sc[k][1] = c.value_scale[scale];
          } else if (at.page == -1) {
            static_cast<uint4*>(a.key)[to] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.tail_k) + off);
            static_cast<uint4*>(a.value)[to] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(c.tail_v) + off);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        if (page[k] < 0) continue;
        const int64_t to = (r0 + r + k * at_once) * vecs + v;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float4 p = dev::decode4<kCode>(w[k][x].x), q = dev::decode4<kCode>(w[k][x].y);
          const float s = sc[k][x];
          static_cast<uint4*>(x ? a.value : a.key)[to] =
              make_uint4(dev::from_f2<kBf16>(p.x * s, p.y * s), dev::from_f2<kBf16>(p.z * s, p.w * s),
                         dev::from_f2<kBf16>(q.x * s, q.y * s), dev::from_f2<kBf16>(q.z * s, q.w * s));
        }
      }
    }
  }
}

template <bool kBf16, int kCode>
int launch(const KittyKv8ReadArgs& a, uint32_t* err, cudaStream_t s) {
  // Many rows: 32 a CTA, which finds their pages once (16 x 32768 tokens of 8 heads of 128: 505 us
  // in a burst and 509 at the clocks of the power cap, with 8 rows 499 and 531; of one head 174,
  // with 8 rows 446).  Few: 8, so that every SM has some (one entry of 4137 tokens 8.9 us, 15.4
  // with 32).
  if (int64_t(a.rows) * a.cache.num_heads * a.cache.head_dim > kManyValues * sm_count())
    return launch_dependent("kv8_read", read_kernel<kBf16, kCode, 32>, dim3(unsigned((int64_t(a.rows) + 31) / 32)),
                            kThreads, 0, s, a, err);
  return launch_dependent("kv8_read", read_kernel<kBf16, kCode, 8>, dim3(unsigned((int64_t(a.rows) + 7) / 8)), kThreads, 0,
                          s, a, err);
}

}  // namespace
}  // namespace kitty8

using namespace kitty8;

extern "C" int kitty_kv8_read(const KittyKv8ReadArgs* a, void* stream) {
  const char* what = "kv8_read";
  if (!a) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "args is NULL");
  const int rc = check_cache(&a->cache, what);
  if (rc != KITTY_OK) return rc;
  if (a->n < 0 || a->rows < 0) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "negative size");
  if (a->n > 0x7fffff00) return fail(KITTY_ERR_UNSUPPORTED, what, "too many entries");     // n + 32 is an int
  if (a->n == 0 || a->rows == 0) return KITTY_OK;
  if (!a->key || !a->value || !a->row_offsets)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "NULL key, value or row_offsets");
  if (!aligned(a->key, 16) || !aligned(a->value, 16))
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "key and value must be 16-byte aligned");
  if (!a->seq_map && a->n > a->cache.slots)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "more entries than slots");
  uint32_t* err = error_word();
  if (!err) return fail(KITTY_ERR_CUDA, what, "no CUDA device");
  cudaStream_t s = as_stream(stream);
  if (a->cache.dtype == KITTY_KV8_BF16)
    return a->cache.code == KITTY_KV8_E4M3 ? launch<true, KITTY_KV8_E4M3>(*a, err, s)
                                           : launch<true, KITTY_KV8_INT8>(*a, err, s);
  return a->cache.code == KITTY_KV8_E4M3 ? launch<false, KITTY_KV8_E4M3>(*a, err, s)
                                         : launch<false, KITTY_KV8_INT8>(*a, err, s);
}
