// Error reporting, struct sizes and the checks that the 8-bit cache entry points share.
#include "kv8_common.cuh"

namespace kitty8 {

__device__ uint32_t g_error = 0;

namespace {
constexpr int kMaxDevices = 64;
thread_local char g_message[256] = "";
}  // namespace

int fail(int code, const char* what, const char* msg) {
  snprintf(g_message, sizeof(g_message), "%s: %s", what, msg);
  return code;
}

int check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? KITTY_OK : fail(KITTY_ERR_CUDA, what, cudaGetErrorString(e));
}

int sm_count() {
  static std::atomic<int> known[kMaxDevices];     // 0: not asked yet
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return 148; }
  if (dev < kMaxDevices && known[dev]) return known[dev];
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
    cudaGetLastError();
    return 148;
  }
  if (dev < kMaxDevices) known[dev] = sms;
  return sms;
}

uint32_t* error_word() {
  static std::atomic<void*> known[kMaxDevices];   // the symbol's address on each device, fixed for the process
  int dev = 0;
  void* p = nullptr;
  if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return nullptr; }
  if (dev < kMaxDevices && known[dev]) return static_cast<uint32_t*>(known[dev].load());
  if (cudaGetSymbolAddress(&p, g_error) != cudaSuccess) { cudaGetLastError(); return nullptr; }
  if (dev < kMaxDevices) known[dev] = p;
  return static_cast<uint32_t*>(p);
}

int check_cache(const KittyKv8Cache* c, const char* what) {
  if (c->num_heads <= 0 || c->head_dim <= 0 || c->page_size <= 0 || c->slots < 0 || c->max_pages < 0 || c->pages < 0 ||
      c->bt_s_slot < 0)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "negative or zero size");
  if (c->head_dim % 16 || c->head_dim > 256)
    return fail(KITTY_ERR_UNSUPPORTED, what, "head_dim must be a multiple of 16 and at most 256");
  if (c->page_size % 32 || c->page_size > 256)
    return fail(KITTY_ERR_UNSUPPORTED, what, "page_size must be a multiple of 32 and at most 256");
  if (c->num_heads > 65535) return fail(KITTY_ERR_UNSUPPORTED, what, "more than 65535 heads");
  if (c->code != KITTY_KV8_E4M3 && c->code != KITTY_KV8_INT8)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "code must be KITTY_KV8_E4M3 or KITTY_KV8_INT8");
  if (c->dtype != KITTY_KV8_F16 && c->dtype != KITTY_KV8_BF16)
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "dtype must be KITTY_KV8_F16 or KITTY_KV8_BF16");
  if (c->pages > 0x7fffffffLL) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "pages must fit int32 page numbers");
  if (c->slots > 0 && (!c->lengths || !c->tail_k || !c->tail_v))
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "NULL lengths or tails");
  if (c->pages > 0 && (!c->key_codes || !c->value_codes || !c->key_scale || !c->value_scale))
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "NULL pools");
  if (c->max_pages > 0 && !c->block_table) return fail(KITTY_ERR_INVALID_ARGUMENT, what, "NULL block table");
  if (!aligned(c->key_codes, 16) || !aligned(c->value_codes, 16) || !aligned(c->tail_k, 16) || !aligned(c->tail_v, 16))
    return fail(KITTY_ERR_INVALID_ARGUMENT, what, "pools and tails must be 16-byte aligned");
  return KITTY_OK;
}

}  // namespace kitty8

using namespace kitty8;

extern "C" {

int kitty_kv8_abi_version(void) { return KITTY_KV8_ABI_VERSION; }

const char* kitty_kv8_last_error(void) { return g_message; }

size_t kitty_kv8_args_size(int kind) {
  switch (kind) {
    case 0: return sizeof(KittyKv8Cache);
    case 1: return sizeof(KittyKv8WriteArgs);
    case 2: return sizeof(KittyKv8ReadArgs);
    case 3: return sizeof(KittyKv8AttentionArgs);
    case 4: return sizeof(KittyQkNormRopeArgs);
    default: return 0;
  }
}

int kitty_kv8_error_flags(uint32_t* flags, int clear) {
  if (!flags) return fail(KITTY_ERR_INVALID_ARGUMENT, "kv8_error_flags", "flags is NULL");
  uint32_t v = 0;
  const uint32_t zero = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, g_error, sizeof(v));
  if (e == cudaSuccess && clear && v) e = cudaMemcpyToSymbol(g_error, &zero, sizeof(zero));
  if (e != cudaSuccess) return fail(KITTY_ERR_CUDA, "kv8_error_flags", cudaGetErrorString(e));
  *flags = v;
  return KITTY_OK;
}

}  // extern "C"
