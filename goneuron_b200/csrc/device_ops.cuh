// device_ops.cuh -- what the operators on device memory share: types, launches on the caller's stream, the status word.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "op_rules.cuh"

namespace gn {

// What kernels of these operators found wrong, one bit each.  Part of the library image and not of a context: a captured graph may be replayed
// after the context that it was captured with is gone.
enum OpStatusBit { OP_BAD_INDEX = 1, OP_TIMEOUT = 2 };
static __device__ int op_status_word;
__device__ __forceinline__ void op_report(int bit) { atomicOr(&op_status_word, bit); }

// Makes the context's GPU the current one for as long as the call takes.
struct OnDevice {
  int was = -1; cudaError_t error;
  explicit OnDevice(int dev) { error = cudaGetDevice(&was); if (error == cudaSuccess && was != dev) error = cudaSetDevice(dev); else was = -1; }
  ~OnDevice() { if (was >= 0) cudaSetDevice(was); }
};
#define GN_OP_BEGIN(name, wrong)                                                                                   \
  if (!ctx || !ctx->alive) return fail(GN_ERR_INVALID_ARG, name ": context is null or shut down");                  \
  if (const char* e_ = (wrong)) return fail(GN_ERR_INVALID_ARG, name ": %s", e_);                                   \
  OnDevice on_device(ctx->c.device);                                                                               \
  if (on_device.error != cudaSuccess) return fail(GN_ERR_CUDA, name ": %s", cudaGetErrorString(on_device.error))

// Launches that touch nothing of the context (GN_LAUNCH counts, and records into a step that another thread may be putting together).  A kernel may be placed while the one before it in the
// stream still runs, whoever launched that: every kernel of these operators calls op_begin() in all threads before it touches global memory, and lets its own successor in there.  (The
// six launches of a feed-forward block's training pass over 333 tokens: 70 -> 62 us.)
__device__ __forceinline__ void op_begin() { pdl_launch(); pdl_wait(); }
template <class... P, class... A>
inline int op_launch(const char* what, void* stream, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, int cluster, A&&... args) {
  cudaLaunchConfig_t cfg{}; cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[2]; int n = 0;
  at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization; at[n++].val.programmaticStreamSerializationAllowed = 1;
  if (cluster > 1) { at[n].id = cudaLaunchAttributeClusterDimension; at[n].val.clusterDim.x = cluster; at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1; n++; }
  cfg.attrs = at; cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  if (e != cudaSuccess) { cudaGetLastError(); return fail(GN_ERR_CUDA, "kernel launch failed (%s): %s", what, cudaGetErrorString(e)); }
  return GN_OK;
}
// The kernel's limit of dynamic shared memory on this GPU.  It belongs to the kernel and not to a launch: every call that needs it sets the most that any call may ask for, so that no thread lowers it between
// another one's setting it and launching.
template <class K> inline int op_smem(const char* what, K kernel, int bytes) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  return e == cudaSuccess ? GN_OK : fail(GN_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// A load from global memory, for whatever these kernels read.  A kernel is there while the ones before it still write, its own operator's earlier launches among them (op_begin), so that nothing is constant
// for as long as it runs: loads of the read-only path, by name or by a const pointer without aliases, would be free to return what memory held before the wait.  Loads of this form stay where they are written,
// side by side (plain ones, moved by the compiler behind what earlier ones decide: 187 instead of 182 us for lookup and gradient of 131072 tokens of 1024, bf16).
template <class T> __device__ __forceinline__ T ld(const T* p) {
  static_assert(sizeof(T) == 4 || sizeof(T) == 8 || sizeof(T) == 16, "");
  T v;
  if constexpr (sizeof(T) == 4) { uint32_t u; asm volatile("ld.global.u32 %0, [%1];" : "=r"(u) : "l"(p)); memcpy(&v, &u, 4); }
  else if constexpr (sizeof(T) == 8) { uint2 u; asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "l"(p)); memcpy(&v, &u, 8); }
  else { uint4 u; asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p)); memcpy(&v, &u, 16); }
  return v;
}

// ------------------------------------------------------------------ elements
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ float2 unpack2(uint32_t u, __half) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
__device__ __forceinline__ float2 unpack2(uint32_t u, __nv_bfloat16) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
// 16 bytes of T as floats, and back (rounded once)
template <class T> struct Vec { static constexpr int N = 16 / sizeof(T); };
template <class T> __device__ __forceinline__ void unpack(const uint4& u, float (&v)[Vec<T>::N]) {
  if constexpr (sizeof(T) == 4) { v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w); }
  else {
    const float2 a = unpack2(u.x, T()), b = unpack2(u.y, T()), c = unpack2(u.z, T()), d = unpack2(u.w, T());
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
}
template <class T> __device__ __forceinline__ uint4 pack(const float (&v)[Vec<T>::N]) {
  if constexpr (sizeof(T) == 4) return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else return make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
}
// two floats an instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r; asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y)); return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r; asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y)); return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r; asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y)); return r;
}
__device__ __forceinline__ int64_t load_index(const void* p, int index_type, int64_t i) {
  return index_type == GN_I64 ? ld(reinterpret_cast<const long long*>(p) + i) : (int64_t)ld(reinterpret_cast<const int*>(p) + i);
}
// Calls f with a value of the type that `dtype` names.
template <class F> inline int with_type(int dtype, F&& f) {
  return dtype == GN_F32 ? f(float()) : dtype == GN_F16 ? f(__half()) : f(__nv_bfloat16());
}

}  // namespace gn
