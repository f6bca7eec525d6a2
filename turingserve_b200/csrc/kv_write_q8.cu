// Rotary positions on queries and keys, and keys and values into an 8-bit paged cache (q8_cache.cuh).
//
// Semantics as rope_kv_write (elementwise.cu): rotate-half over the first `rot` dims of each query and key head with the
// table's rows rounded to the model's type and the arithmetic in 32 bits; slot < 0 writes nothing.  What differs: the
// rotated queries go to `q_out` and qkv stays as it was (every block of rows reads its neighbours' keys for their page's
// largest value, so nothing may be turned in place), and the cache takes round_e4m3(x / s) with x the rotated key in 32
// bits (not rounded to the model's type first) or the value, and s the page's scale for that kv head:
//   s = the least power of two under which the rows fit, and, unless one of the rows is the page's first, not below the
//       scale that the page had; when it grows, the page's other rows are brought to it.
// A page's rows stand next to each other among the tokens that are written (a request's tokens do); no slot appears twice.
#include "q8_cache.cuh"

namespace {

using namespace q8;

struct WriteArgs {
  const void* qkv;
  void* q_out;
  long long q_stride;                 // elements between rows of q_out
  const int* positions;
  const float* cos_t;
  const float* sin_t;
  unsigned char* cache[2];            // keys, values
  float* scale[2];
  const int* slots;
  int T, H, KVH, D, rot, page;
};

template <typename T>
__device__ __forceinline__ float rotated(const T* x, int d, int rot, const float* cos_row, const float* sin_row) {
  const int half = rot / 2;
  if (d >= rot) return to_f(x[d]);
  const int i = d < half ? d : d - half;
  const float c = round_to<T>(cos_row[i]), s = round_to<T>(sin_row[i]);
  const float a = to_f(x[i]), b = to_f(x[i + half]);
  return d < half ? a * c - b * s : b * c + a * s;
}

// Any sizes: block (token, head).  A query head is turned; for a key or value head the block of a page's first token among the
// tokens writes all of the page's rows, the others have nothing to do.
template <typename T>
__global__ void kv_write_q8_kernel(const WriteArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x, D = a.D, heads = a.H + 2 * a.KVH;
  const T* qkv = (const T*)a.qkv;
  if ((int)blockIdx.y < a.H) {
    const int h = blockIdx.y, pos = a.positions[t];
    const T* x = qkv + ((size_t)t * heads + h) * D;
    const float* c = a.cos_t + (size_t)pos * (a.rot / 2);
    const float* s = a.sin_t + (size_t)pos * (a.rot / 2);
    T* o = (T*)a.q_out + (size_t)t * a.q_stride + (size_t)h * D;
    for (int d = threadIdx.x; d < D; d += blockDim.x) o[d] = from_f<T>(rotated(x, d, a.rot, c, s));
    return;
  }
  const int kv = (blockIdx.y - a.H) / a.KVH, kvh = (blockIdx.y - a.H) % a.KVH;       // keys or values; which kv head
  const int slot = a.slots[t];
  if (slot < 0) return;
  const int pg = slot / a.page;
  int before = t - 1;
  while (before >= 0 && a.slots[before] < 0) --before;
  if (before >= 0 && a.slots[before] / a.page == pg) return;
  int end = t + 1;
  bool anew = slot % a.page == 0;
  for (int u = end; u < a.T; ++u) {
    const int s = a.slots[u];
    if (s < 0) continue;
    if (s / a.page != pg) break;
    anew = anew || s % a.page == 0;
    end = u + 1;
  }

  auto value = [&](int row, int d) {
    const T* x = qkv + ((size_t)row * heads + a.H + kv * a.KVH + kvh) * D;
    if (kv) return to_f(x[d]);
    const size_t at = (size_t)a.positions[row] * (a.rot / 2);
    return rotated(x, d, a.rot, a.cos_t + at, a.sin_t + at);
  };
  __shared__ unsigned amax_s;
  if (threadIdx.x == 0) amax_s = 0;
  __syncthreads();
  unsigned amax = 0;
  const int total = (end - t) * D;
  for (int i = threadIdx.x; i < total; i += blockDim.x)
    if (a.slots[t + i / D] >= 0) amax = max(amax, __float_as_uint(fabsf(value(t + i / D, i % D))));
  atomicMax(&amax_s, amax);
  float* sp = a.scale[kv] + (size_t)pg * a.KVH + kvh;
  const float held = *sp;
  __syncthreads();
  const float need = scale_for(amax_s), now = anew ? need : larger_scale(held, need), inv = inverse_scale(now);
  unsigned char* rows = a.cache[kv] + ((size_t)pg * a.KVH + kvh) * a.page * D;
  if (!anew && now > held) {                                                         // (a NaN compares false: nothing to bring)
    const float ratio = held * inv;
    for (int r = 0; r < a.page; ++r) {
      bool written = false;
      for (int u = t; u < end; ++u) written = written || (a.slots[u] >= 0 && a.slots[u] % a.page == r);
      if (written) continue;
      for (int d = threadIdx.x; d < D; d += blockDim.x) rows[(size_t)r * D + d] = to_e4m3(from_e4m3(rows[(size_t)r * D + d]) * ratio);
    }
  }
  for (int i = threadIdx.x; i < total; i += blockDim.x) {
    const int row = t + i / D, d = i % D;
    if (a.slots[row] >= 0) rows[(size_t)(a.slots[row] % a.page) * D + d] = quantise(value(row, d), inv);
  }
  if (threadIdx.x == 0) *sp = now;
}

}  // namespace

// qkv [T, (H + 2 KVH) * D], q_out [T, H * D] with rows q_stride elements apart.  k_cache null: queries only.
TS_API int ts_rope_kv_write_q8(void* q_out, long long q_stride, const void* qkv, const int* positions, const float* cos_t,
                               const float* sin_t, void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                               const int* slots, int T, int H, int KVH, int D, int rot, int page, int dtype, void* stream) {
  if (T <= 0) return 0;
  if (H <= 0 || KVH <= 0 || D <= 0 || page <= 0 || H + 2 * KVH > 65535)
    TS_REFUSE(TS_ERR_SHAPE, "ts_rope_kv_write_q8: H=%d KVH=%d D=%d page=%d", H, KVH, D, page);
  if (rot < 0 || rot > D || (rot & 1)) TS_REFUSE(TS_ERR_SHAPE, "ts_rope_kv_write_q8: rotary_dim %d for head_dim %d", rot, D);
  if (rot > 0 && (cos_t == nullptr || sin_t == nullptr)) TS_REFUSE(TS_ERR_SHAPE, "ts_rope_kv_write_q8: tables missing");
  if (k_cache != nullptr && (v_cache == nullptr || k_scale == nullptr || v_scale == nullptr || slots == nullptr))
    TS_REFUSE(TS_ERR_SHAPE, "ts_rope_kv_write_q8: keys without values, scales or slots");
  if (dtype != TS_F32 && dtype != TS_BF16) TS_REFUSE(TS_ERR_DTYPE, "ts_rope_kv_write_q8: dtype %d", dtype);
  WriteArgs a = {qkv, q_out, q_stride, positions, cos_t, sin_t, {(unsigned char*)k_cache, (unsigned char*)v_cache},
                 {k_scale, v_scale}, slots, T, H, KVH, D, rot, page};
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid(T, k_cache != nullptr ? H + 2 * KVH : H), block(D >= 128 ? 128 : 64);
  if (dtype == TS_F32) ts_launch(kv_write_q8_kernel<float>, grid, block, 0, s, a);
  else ts_launch(kv_write_q8_kernel<bf16>, grid, block, 0, s, a);
  TS_LAUNCH_CHECK();
}
