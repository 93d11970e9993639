// Reading the cache back to 16-bit rows.
//
// A CTA takes kRows output rows (tokens, all heads).  Its first warp finds each row's slot
// and page by a search of the row offsets and leaves them in shared memory; then every
// thread turns eight codes of keys and of values (8 bytes each) into 16-byte stores,
// contiguous over the row, at the same place of one row after another.  Bound by HBM: 1
// byte read and 2 written a value.
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
  if (int(threadIdx.x) < count) {
    const int r = int(r0) + threadIdx.x;
    int lo = 0, hi = a.n + 1;            // how many offsets are <= r (any contents end within the bounds)
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.row_offsets[mid] <= r) lo = mid + 1;
      else hi = mid;
    }
    const int i = lo - 1;
    RowAt at{0, -2};
    uint32_t bad = 0;
    if (i >= 0 && i < a.n) {
      const int slot = a.seq_map ? a.seq_map[i] : i;
      const int64_t first = a.first ? a.first[i] : 0;
      const int o = a.row_offsets[i];
      if (o < 0 || o > r) {
        bad = kErrRows;
      } else if (slot >= c.slots) {
        bad = kErrSlot;
      } else if (slot >= 0) {                 // (a negative slot is padding)
        const int64_t t = first + (r - o);
        const int len = c.lengths[slot];
        if (t < 0 || t >= len || len / G > c.max_pages) {
          bad = kErrLength;
        } else {
          const int b = int(t / G), in = int(t % G);
          if (b < len / G) {
            const int page = c.block_table[int64_t(slot) * c.bt_s_slot + b];
            if (page < 0 || page >= c.pages) bad = kErrPage;
            else at = RowAt{(int64_t(page) * H * G + in) * D, page};
          } else {
            at = RowAt{(int64_t(slot) * H * G + in) * D, -1};
          }
        }
      }
    }
    if (bad) dev::flag(err, bad);
    s_row[threadIdx.x] = at;
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
  // Many rows: 32 a CTA, which finds their pages once.  Few: 8, so that every SM has some.
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
