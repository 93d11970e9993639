// RMS norm of every query and key head with the rotary embedding in the same pass.
//
// A row (one head of one token, D channels) is held by the lanes of a group: the lane
// that rotates pairs 8j .. 8j+7 has all sixteen values of those pairs in registers
// (two 16-byte loads), so the rotation needs no exchange and the mean of squares one
// butterfly over the group.  A warp keeps its token's cosines and sines over up to
// kPasses rows per group.  It is bound by HBM, 2 bytes read and 2 written a channel, and
// what is in flight counts: a warp's next token is copied to shared memory while this one
// is worked on.  Every thread reads back only what it copied itself, so nothing is
// synchronised.
#include "kv8_common.cuh"

namespace kitty8 {
namespace {

constexpr int kThreads = 256;
// CTAs resident on an SM: a warp with one row for each lane group needs half the registers and
// has a quarter of the bytes in flight.
template <int kPasses>
constexpr int kCtas = kPasses == 1 ? 3 : 2;

struct RopeShape {
  int q_chunks, chunks;        // warps per token: ceil(heads / rows of a warp), queries first
};

__device__ __forceinline__ void copy_async(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
               :: "r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}

// kPasses: rows per lane group and token, which share the table values; kStages: tokens of
// a warp in flight in shared memory, 0: no stage, the rows go to registers.
template <bool kBf16, int kLanes, bool kInter, int kPasses, int kStages>
__global__ void __launch_bounds__(kThreads, kCtas<kPasses>) qk_norm_rope_kernel(KittyQkNormRopeArgs a, RopeShape sh, uint32_t* err) {
  constexpr int kRows = 32 / kLanes;                       // rows that a warp holds at once
  dev::wait_for_stream();
  const int lane = threadIdx.x & 31, j = lane % kLanes;
  const int64_t warps = int64_t(gridDim.x) * (kThreads / 32) / sh.chunks * sh.chunks;
  const int64_t gw = int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (gw >= warps) return;
  const int chunk = int(gw % sh.chunks);                   // the same heads for every token of this warp
  const bool is_q = chunk < sh.q_chunks;
  const int heads = is_q ? a.num_q_heads : a.num_k_heads;
  const int h0 = (is_q ? chunk : chunk - sh.q_chunks) * (kRows * kPasses) + lane / kLanes;
  const int D = a.head_dim, pair_lanes = a.rot / 16;
  const bool active = j < D / 16, rotates = j < pair_lanes;
  // first channel of the lane's two groups of eight
  int c0, c1;
  if (kInter || !rotates) {
    c0 = rotates ? 16 * j : a.rot + 16 * (j - pair_lanes);
    c1 = c0 + 8;
  } else {
    c0 = 8 * j;
    c1 = c0 + a.rot / 2;
  }
  const uint16_t* in = static_cast<const uint16_t*>(is_q ? a.q : a.k);
  uint16_t* out = static_cast<uint16_t*>(is_q ? a.q_out : a.k_out);
  const int64_t s_row = is_q ? a.q_s_row : a.k_s_row, s_head = is_q ? a.q_s_head : a.k_s_head;
  const int64_t o_row = is_q ? a.qo_s_row : a.ko_s_row, o_head = is_q ? a.qo_s_head : a.ko_s_head;
  const void* wp = is_q ? a.q_weight : a.k_weight;
  float w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = (i < 8 ? c0 : c1 - 8) + i;
    w[i] = 1.f;
    if (wp && active) {
      if (a.weight_f32) w[i] = static_cast<const float*>(wp)[c];
      else w[i] = dev::to_f2<kBf16>(static_cast<const uint16_t*>(wp)[c]).x;
    }
  }
  const float inv_d = 1.f / float(D);
  // [stage][warp][pass][half][lane]
  extern __shared__ uint4 s_x[];
  uint4* const mine = s_x + (threadIdx.x >> 5) * (kPasses * 2 * 32) + lane;
  [[maybe_unused]] constexpr int kStage = (kThreads / 32) * kPasses * 2 * 32;
  const int64_t step = warps / sh.chunks;
  uint4 direct[kStages ? 1 : kPasses * 2];
  auto fetch = [&](int64_t t, int stage) {
    if (kStages == 0 || (t < a.rows && active)) {
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int h = h0 + p * kRows;
        const uint16_t* r = in + t * s_row + h * s_head;
        if constexpr (kStages > 0) {
          if (h < heads) {
            copy_async(mine + stage * kStage + p * 64, r + c0);
            copy_async(mine + stage * kStage + p * 64 + 32, r + c1);
          }
        } else {
          const bool there = active && h < heads;
          direct[2 * p] = there ? *reinterpret_cast<const uint4*>(r + c0) : make_uint4(0, 0, 0, 0);
          direct[2 * p + 1] = there ? *reinterpret_cast<const uint4*>(r + c1) : make_uint4(0, 0, 0, 0);
        }
      }
    }
    if constexpr (kStages > 0) asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // The copies of the token at hand are there; only the later ones' may be on their way.
  auto arrive = [&]() {
    if constexpr (kStages > 0) asm volatile("cp.async.wait_group %0;" :: "n"(kStages - 1) : "memory");
  };
  auto position = [&](int64_t t) {
    return t >= a.rows ? int64_t(-1)
           : a.positions64 ? static_cast<const int64_t*>(a.positions)[t]
                           : int64_t(static_cast<const int32_t*>(a.positions)[t]);
  };
  int64_t t = gw / sh.chunks;
#pragma unroll
  for (int i = 0; i + 1 < kStages; ++i) fetch(t + i * step, i);
  int64_t next = position(t);                               // read a token ahead: the table waits for it
  for (int stage = 0; t < a.rows; t += step, stage = stage + 1 == kStages ? 0 : stage + 1) {
    const int64_t pos = next;
    next = position(t + step);
    if constexpr (kStages > 0) fetch(t + (kStages - 1) * step, stage == 0 ? kStages - 1 : stage - 1);
    else fetch(t, 0);
    if (pos < 0 || pos >= a.table_rows) {                   // a padding row, or none of the table
      if (pos >= 0 && lane == 0) dev::flag(err, kErrPosition);
      arrive();                                             // before another copy goes to this stage
      continue;
    }
    float cs[8], sn[8];
    if (rotates) {
      const float4* tc = reinterpret_cast<const float4*>(a.table + pos * a.rot + 8 * j);
      const float4* ts = reinterpret_cast<const float4*>(a.table + pos * a.rot + a.rot / 2 + 8 * j);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 u = tc[i], v = ts[i];
        cs[4 * i] = u.x; cs[4 * i + 1] = u.y; cs[4 * i + 2] = u.z; cs[4 * i + 3] = u.w;
        sn[4 * i] = v.x; sn[4 * i + 1] = v.y; sn[4 * i + 2] = v.z; sn[4 * i + 3] = v.w;
      }
    }
    arrive();
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int h = h0 + p * kRows;
      float y[16];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint4 x;
        if constexpr (kStages > 0)
          x = active && h < heads ? mine[stage * kStage + p * 64 + half * 32] : make_uint4(0, 0, 0, 0);
        else
          x = direct[2 * p + half];
        const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = dev::to_f2<kBf16>(u[i]);
          y[8 * half + 2 * i] = f.x;
          y[8 * half + 2 * i + 1] = f.y;
        }
      }
      if (wp) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(y[i], y[i], ss);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float rs = rsqrtf(fmaf(ss, inv_d, a.eps));
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] *= rs * w[i];
      }
      if (rotates) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float& u = y[kInter ? 2 * i : i];
          float& v = y[kInter ? 2 * i + 1 : 8 + i];
          const float ua = u, va = v;
          u = fmaf(ua, cs[i], -(va * sn[i]));
          v = fmaf(va, cs[i], ua * sn[i]);
        }
      }
      if (active && h < heads) {
        uint16_t* r = out + t * o_row + h * o_head;
        *reinterpret_cast<uint4*>(r + c0) =
            make_uint4(dev::from_f2<kBf16>(y[0], y[1]), dev::from_f2<kBf16>(y[2], y[3]),
                       dev::from_f2<kBf16>(y[4], y[5]), dev::from_f2<kBf16>(y[6], y[7]));
        *reinterpret_cast<uint4*>(r + c1) =
            make_uint4(dev::from_f2<kBf16>(y[8], y[9]), dev::from_f2<kBf16>(y[10], y[11]),
                       dev::from_f2<kBf16>(y[12], y[13]), dev::from_f2<kBf16>(y[14], y[15]));
      }
    }
  }
}

template <bool kBf16, int kLanes, int kPasses, int kStages>
int launch(const KittyQkNormRopeArgs& a, uint32_t* err, cudaStream_t s) {
  constexpr int kHeads = 32 / kLanes * kPasses;
  RopeShape sh;
  sh.q_chunks = (a.num_q_heads + kHeads - 1) / kHeads;
  sh.chunks = sh.q_chunks + (a.num_k_heads + kHeads - 1) / kHeads;
  const int64_t warps = int64_t(a.rows) * sh.chunks, per = kThreads / 32;
  // at least one warp for each chunk of heads, at most what the card holds at once
  const int64_t most = std::max<int64_t>(int64_t(sm_count()) * kCtas<kPasses>, (sh.chunks + per - 1) / per);
  const int64_t grid = std::min((warps + per - 1) / per, most);
  constexpr int kBytes = kStages * (kThreads / 32) * kPasses * 2 * 32 * 16;
  const auto kernel = a.interleaved ? qk_norm_rope_kernel<kBf16, kLanes, true, kPasses, kStages>
                                    : qk_norm_rope_kernel<kBf16, kLanes, false, kPasses, kStages>;
  if (kBytes > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess)
    return check_launch("qk_norm_rope");
  return launch_dependent("qk_norm_rope", kernel, dim3(unsigned(grid)), kThreads, kBytes, s, a, sh, err);
}

template <bool kBf16, int kLanes>
int launch_size(const KittyQkNormRopeArgs& a, uint32_t* err, cudaStream_t s) {
  // Stages pay where a resident warp has more than one token (40 heads of 128: 6.1 against
  // 6.4 us for 1024 tokens, 31 against 38 for 8192, 111 against 136 for 32768) and cost where it
  // has one (301 tokens of 72 heads: 5.6 and 4.6 us).
  // With no more heads than a warp has lane groups, rows behind the first would be empty.
  if (std::max(a.num_q_heads, a.num_k_heads) <= 32 / kLanes) return launch<kBf16, kLanes, 1, 0>(a, err, s);
  constexpr int kStaged = 4, kHeads = 32 / kLanes * kStaged;
  const int64_t chunks = (a.num_q_heads + kHeads - 1) / kHeads + (a.num_k_heads + kHeads - 1) / kHeads;
  return a.rows * chunks > int64_t(sm_count()) * kCtas<kStaged> * (kThreads / 32) ? launch<kBf16, kLanes, kStaged, 2>(a, err, s)
                                                                         : launch<kBf16, kLanes, 2, 0>(a, err, s);
}

template <bool kBf16>
int launch_dim(const KittyQkNormRopeArgs& a, uint32_t* err, cudaStream_t s) {
  if (a.head_dim <= 64) return launch_size<kBf16, 4>(a, err, s);
  if (a.head_dim <= 128) return launch_size<kBf16, 8>(a, err, s);
  return launch_size<kBf16, 16>(a, err, s);
}

}  // namespace
}  // namespace kitty8

using namespace kitty8;

extern "C" int kitty_qk_norm_rope(const KittyQkNormRopeArgs* a, void* stream) {
  const char* what = "qk_norm_rope";
  if (!a) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "args is NULL");
  if (a->rows < 0 || a->num_q_heads < 0 || a->num_k_heads < 0 || a->head_dim <= 0 || a->rot < 0 || a->table_rows < 0)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "negative or zero size");
  if (a->head_dim % 16 || a->head_dim > 256)
    return fail(KITTY_ERR_UNSUPPORTED, what, "head_dim must be a multiple of 16 and at most 256");
  if (a->rot % 16 || a->rot > a->head_dim)
    return fail(KITTY_ERR_UNSUPPORTED, what, "the rotary width must be a multiple of 16 and at most head_dim");
  if (a->dtype != KITTY_KV8_F16 && a->dtype != KITTY_KV8_BF16)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "dtype must be KITTY_KV8_F16 or KITTY_KV8_BF16");
  if ((a->q_weight == nullptr) != (a->k_weight == nullptr))
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "q_weight and k_weight go together");
  if (a->rows == 0 || a->num_q_heads + a->num_k_heads == 0) return KITTY_OK;
  if (!a->positions || (a->rot > 0 && !a->table)) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "NULL positions or table");
  if ((a->num_q_heads > 0 && (!a->q || !a->q_out)) || (a->num_k_heads > 0 && (!a->k || !a->k_out)))
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "NULL q, k or outputs");
  const int64_t strides[] = {a->q_s_row, a->q_s_head, a->k_s_row, a->k_s_head,
                             a->qo_s_row, a->qo_s_head, a->ko_s_row, a->ko_s_head};
  for (int64_t v : strides)
    if (v % 8) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "row and head strides must be multiples of 8 elements");
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->q_out, 16) || !aligned(a->k_out, 16) ||
      !aligned(a->table, 16))
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "tensors must be 16-byte aligned");
  uint32_t* err = error_word();
  if (!err) return fail(KITTY_ERR_CUDA, what, "no CUDA device");
  return a->dtype == KITTY_KV8_BF16 ? launch_dim<true>(*a, err, as_stream(stream))
                                    : launch_dim<false>(*a, err, as_stream(stream));
}
