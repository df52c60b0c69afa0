// C ABI of the AdamW step (declared in include/avey_b200.h): argument checks,
// the tables of tensors and the launches of adamw_kernels.cuh.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "avey_b200.h"
#include "host_api.h"
#include "adamw_kernels.cuh"

namespace {

int fail(int code, const char* msg) { return avey_host::set_error(code, msg); }

// Tensors per launch: 400 entries of 80 bytes fit the 32,764 bytes of kernel
// parameters; calls of up to 48 tensors pass a table of that size instead.
constexpr int kMany = 400, kFew = 48;

constexpr int kMaxDevices = 64;

// Opt kernel K into its shared memory, once per device; the outcome is kept.
template <auto K>
cudaError_t smem_opt_in(int bytes) {
  static std::once_flag once[kMaxDevices];
  static cudaError_t err[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [dev, bytes] {
    err[dev] = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  });
  return err[dev];
}

int validate(const AveyAdamWParams* p) {
  if (!p) return fail(AVEY_ERR_ARGUMENT, "params is NULL");
  if (p->struct_size != sizeof(AveyAdamWParams))
    return fail(AVEY_ERR_ARGUMENT, "struct_size does not match sizeof(AveyAdamWParams)");
  if (p->dtype != AVEY_F32 && p->dtype != AVEY_F16 && p->dtype != AVEY_BF16)
    return fail(AVEY_ERR_ARGUMENT, "adamw takes f32, f16 or bf16 parameters");
  if (p->state_bits != 32 && p->state_bits != 8) return fail(AVEY_ERR_ARGUMENT, "state_bits must be 32 or 8");
  if (p->count < 0 || (p->count > 0 && !p->tensors)) return fail(AVEY_ERR_ARGUMENT, "tensors is required");
  if (!std::isfinite(p->lr) || p->lr < 0 || !std::isfinite(p->weight_decay) || p->weight_decay < 0 ||
      !std::isfinite(p->eps) || p->eps < 0)
    return fail(AVEY_ERR_ARGUMENT, "lr, eps and weight_decay must be finite and not negative");
  if (!(p->beta1 >= 0 && p->beta1 < 1 && p->beta2 >= 0 && p->beta2 < 1))
    return fail(AVEY_ERR_ARGUMENT, "beta1 and beta2 must be in [0, 1)");
  if (p->step < 1) return fail(AVEY_ERR_ARGUMENT, "step must be at least 1");
  for (int i = 0; i < p->count; ++i) {
    const AveyAdamWTensor& t = p->tensors[i];
    if (t.numel < 0) return fail(AVEY_ERR_ARGUMENT, "numel must not be negative");
    if (t.numel == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq)
      return fail(AVEY_ERR_ARGUMENT, "param, grad, exp_avg and exp_avg_sq are required");
    if (p->state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale))
      return fail(AVEY_ERR_ARGUMENT, "8-bit states need exp_avg_scale and exp_avg_sq_scale");
    auto bits = [](const void* a) { return reinterpret_cast<uintptr_t>(a); };
    const uintptr_t value = (bits(t.param) | bits(t.grad)) & (p->dtype == AVEY_F32 ? 3u : 1u);
    uintptr_t word = bits(t.master) | bits(t.exp_avg_scale) | bits(t.exp_avg_sq_scale);
    if (p->state_bits == 32) word |= bits(t.exp_avg) | bits(t.exp_avg_sq);
    if (value != 0 || (word & 3u) != 0) return fail(AVEY_ERR_ARGUMENT, "arrays must be aligned to their elements");
  }
  return AVEY_OK;
}

template <typename T, bool MASTER, bool Q8, int N>
int launch(const AveyAdamWTensor* t, int count, int64_t* block0, const avey::AwScalars& c, cudaStream_t stream) {
  avey::AwTable<N> tab;
  tab.count = 0;
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    if (t[i].numel == 0) continue;
    avey::AwTensor& e = tab.t[tab.count++];
    e.p = t[i].param;
    e.g = t[i].grad;
    e.m = t[i].exp_avg;
    e.v = t[i].exp_avg_sq;
    e.ms = t[i].exp_avg_scale;
    e.vs = t[i].exp_avg_sq_scale;
    e.master = t[i].master;
    e.n = t[i].numel;
    e.block0 = *block0;
    e.chunk0 = static_cast<int32_t>(chunks);
    uintptr_t at = (reinterpret_cast<uintptr_t>(e.p) | reinterpret_cast<uintptr_t>(e.g)) & (8 * sizeof(T) - 1);
    at |= (reinterpret_cast<uintptr_t>(e.m) | reinterpret_cast<uintptr_t>(e.v)) & 7u;
    if (MASTER) at |= reinterpret_cast<uintptr_t>(e.master) & 31u;
    e.whole = at == 0 ? static_cast<int32_t>(t[i].numel / avey::kAwChunk) : 0;
    *block0 += (t[i].numel + avey::kAwBlock - 1) / avey::kAwBlock;
    chunks += (t[i].numel + avey::kAwChunk - 1) / avey::kAwChunk;
    if (chunks > (1 << 30)) return fail(AVEY_ERR_ARGUMENT, "more than 2^41 elements in a launch");
  }
  tab.chunks = static_cast<int>(chunks);
  if (tab.chunks == 0) return AVEY_OK;
  const int64_t sms = avey_host::multiprocessors();
  if constexpr (Q8) {
    const int grid = static_cast<int>(std::min<int64_t>(tab.chunks, sms * avey::kAwCtas8));
    constexpr int smem = avey::kAwStages * sizeof(avey::AwStage<T, MASTER>);
    const cudaError_t attr = smem_opt_in<avey::adamw8_step<T, MASTER, N>>(smem);
    if (attr != cudaSuccess) return fail(AVEY_ERR_CUDA, cudaGetErrorString(attr));
    avey::adamw8_step<T, MASTER, N><<<grid, avey::kAwThreads, smem, stream>>>(tab, c);
  } else {
    const int grid = static_cast<int>(std::min<int64_t>(tab.chunks, sms * 8));
    avey::adamw_step<T, MASTER, N><<<grid, avey::kAwThreads, 0, stream>>>(tab, c);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(AVEY_ERR_LAUNCH, cudaGetErrorString(e));
  avey_host::count_launches(1);
  return AVEY_OK;
}

template <typename T, bool MASTER, bool Q8>
int run(const AveyAdamWParams* p, const avey::AwScalars& c, cudaStream_t stream) {
  int64_t block0 = 0;
  for (int i = 0; i < p->count; i += kMany) {
    const int n = std::min(kMany, p->count - i);
    const int rc = n <= kFew ? launch<T, MASTER, Q8, kFew>(p->tensors + i, n, &block0, c, stream)
                             : launch<T, MASTER, Q8, kMany>(p->tensors + i, n, &block0, c, stream);
    if (rc != AVEY_OK) return rc;
  }
  return avey_host::clear_error();
}

template <typename T>
int run_type(const AveyAdamWParams* p, const avey::AwScalars& c, bool master, cudaStream_t s) {
  if (p->state_bits == 8) return master ? run<T, true, true>(p, c, s) : run<T, false, true>(p, c, s);
  return master ? run<T, true, false>(p, c, s) : run<T, false, false>(p, c, s);
}

}  // namespace

extern "C" int avey_adamw_v1(const AveyAdamWParams* p, void* stream) {
  int rc = validate(p);
  if (rc != AVEY_OK) return rc;
  int with = 0, live = 0;
  for (int i = 0; i < p->count; ++i) {
    live += p->tensors[i].numel > 0;
    with += p->tensors[i].numel > 0 && p->tensors[i].master != nullptr;
  }
  if (with != 0 && with != live) return fail(AVEY_ERR_ARGUMENT, "master copies are for all tensors or for none");
  if (live == 0) return avey_host::clear_error();
  rc = avey_host::device_ok();
  if (rc != AVEY_OK) return rc;
  avey::AwScalars c{};
  const double bc1 = 1.0 - std::pow(p->beta1, static_cast<double>(p->step));
  const double bc2 = 1.0 - std::pow(p->beta2, static_cast<double>(p->step));
  c.b1 = static_cast<float>(p->beta1);
  c.c1 = static_cast<float>(1.0 - p->beta1);
  c.b2 = static_cast<float>(p->beta2);
  c.c2 = static_cast<float>(1.0 - p->beta2);
  c.decay = static_cast<float>(1.0 - p->lr * p->weight_decay);
  c.step_size = static_cast<float>(p->lr / bc1);
  c.inv_bc2 = static_cast<float>(1.0 / std::sqrt(bc2));
  c.eps = static_cast<float>(p->eps);
  auto twice = [](float x) { return make_float2(x, x); };
  c.b1p = twice(c.b1);
  c.c1p = twice(c.c1);
  c.b2p = twice(c.b2);
  c.c2p = twice(c.c2);
  c.decayp = twice(c.decay);
  c.minus_stepp = twice(-c.step_size);
  c.inv_bc2p = twice(c.inv_bc2);
  c.epsp = twice(c.eps);
  c.minus_zerop = twice(-0.f);
  c.seed = static_cast<uint32_t>(p->seed);
  c.step = static_cast<uint32_t>(p->step);
  c.key = avey::aw_key(c.seed, c.step, 0);
  c.grad_scale = p->grad_scale;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p->dtype) {
    case AVEY_F32: return run_type<float>(p, c, with > 0, s);
    case AVEY_F16: return run_type<__half>(p, c, with > 0, s);
    default: return run_type<__nv_bfloat16>(p, c, with > 0, s);
  }
}
