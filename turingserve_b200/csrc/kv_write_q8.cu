// Rotary positions on queries and keys, and keys and values into an 8-bit paged cache (q8_cache.cuh).
//
// Semantics as rope_kv_write (elementwise.cu): rotate-half over the first `rot` dims of each query and key head with the
// table's rows rounded to the model's type and the arithmetic in 32 bits; slot < 0 writes nothing.  What differs: the
// rotated queries go to `q_out`, which may not lie in qkv, and qkv stays as it was (every block of rows reads its neighbours' keys for their page's
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

// Any sizes (the float32 path and what the variant below does not take): block (token, head).  A query head is turned; for a key or value head the block of a page's first token among the
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


// bfloat16 heads of 64 or 128, rotated whole or not at all.  A row of a head is D / 16 lanes of 16 values (8 of each half, so that a
// lane turns its own pairs).  A block takes `span` neighbouring tokens.
//   Queries (blockIdx.y >= kv_blocks): some heads of those tokens; a lane keeps its table row for all of them.
//   Keys or values of one kv head: the pages' rows among the tokens, `runs`, reach over the block's edges, so the block reads on to both
//   sides until the first and the last run end: their largest values then are every block's that shares a run, no block waits for
//   another, and all compute the same scale (the scale that a page had is a lower bound: reading it after the run's first
//   block has put the new one there gives the same).  The run's first block brings the page's other rows to a larger scale.
// What bounds it: a few tokens the chain of loads (slots and rows, then the scale: two trips; 1 token of 12 heads over 2 3.4 us in a graph, 64 of
// 28 over 4 5.0), thousands the bytes of qkv once and of the outputs (7,787 tokens of 28 over 4 31 us, 4.5 TB/s of those), the rows
// read twice coming out of L1 or L2.  A decode step of up to 128 tokens brings the product's sums instead (PART): rows of floats, one for each
// split that `linear` left, read again by every block of a run (us, single tokens in pages of 16, finished / sums: 12 heads over 2, 1 token 3.4 / 3.7, 8
// 3.6 / 4.0, 16 4.5 / 5.2, 64 of 6 splits 4.9 / 6.4, 128 of 3 5.0 / 6.1; 28 over 4, 64 of 4 5.0 / 6.0, 128 of 4 5.2 / 6.8; 14 over 2 of 64, 64 of 3
// 4.9 / 5.9), and nothing has to finish the product before it.
constexpr int SPAN_MAX = 64, HEADS = 2;

struct FastArgs {
  WriteArgs w;
  const float* part;                  // [splits][T][(H + 2 KVH) D]: the product's partial sums (null: qkv is finished)
  const bf16* bias;
  int splits;
  int span, kv_blocks, q_heads;
};

// 16 values of a row: 8 at column c1 and 8 at c2 of token t's row of qkv, summed over the splits where it is not finished, and then
// rounded as the product's own end would have rounded them
__device__ __forceinline__ void widen16(const uint4& u, const uint4& v, float (&x)[16]) {
  const unsigned w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <bool PART>
__device__ __forceinline__ void load16(const FastArgs& a, int t, int row_elems, int c1, int c2, float (&x)[16]) {
  if constexpr (!PART) {
    const bf16* r = (const bf16*)a.w.qkv + (size_t)t * row_elems;
    widen16(*reinterpret_cast<const uint4*>(r + c1), *reinterpret_cast<const uint4*>(r + c2), x);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;
    const float* p = a.part + (size_t)t * row_elems;
    const size_t stride = (size_t)a.w.T * row_elems;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p + s * stride + (q < 2 ? c1 : c2 - 8) + 4 * q));
        x[4 * q] += v.x;
        x[4 * q + 1] += v.y;
        x[4 * q + 2] += v.z;
        x[4 * q + 3] += v.w;
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (a.bias != nullptr) x[i] += to_f(a.bias[(i < 8 ? c1 : c2 - 8) + i]);
      x[i] = round_to<bf16>(x[i]);
    }
  }
}
__device__ __forceinline__ void load_table(const WriteArgs& a, int position, int half, int j, float (&c)[8], float (&s)[8]) {
  const size_t at = (size_t)position * half + 8 * j;
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const float4 u = *reinterpret_cast<const float4*>(a.cos_t + at + i), v = *reinterpret_cast<const float4*>(a.sin_t + at + i);
    c[i] = round_to<bf16>(u.x); c[i + 1] = round_to<bf16>(u.y); c[i + 2] = round_to<bf16>(u.z); c[i + 3] = round_to<bf16>(u.w);
    s[i] = round_to<bf16>(v.x); s[i + 1] = round_to<bf16>(v.y); s[i + 2] = round_to<bf16>(v.z); s[i + 3] = round_to<bf16>(v.w);
  }
}
__device__ __forceinline__ void turn(float (&x)[16], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x[i], b = x[8 + i];
    x[i] = a * c[i] - b * s[i];
    x[8 + i] = b * c[i] + a * s[i];
  }
}
__device__ __forceinline__ unsigned four_e4m3(float a, float b, float c, float d) {
  const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

template <int D, int THREADS, bool PART>
__global__ void __launch_bounds__(THREADS) kv_write_q8_fast_kernel(const FastArgs f) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int LPR = D / 16, ROWS = THREADS / LPR, HALF = D / 2;
  const WriteArgs& a = f.w;
  const int tid = threadIdx.x, j = tid % LPR, r = tid / LPR, row_elems = (a.H + 2 * a.KVH) * D;
  const int w0 = blockIdx.x * f.span, w1 = min(a.T, w0 + f.span);
  if ((int)blockIdx.y >= f.kv_blocks) {
    const int h0 = (blockIdx.y - f.kv_blocks) * f.q_heads, h1 = min(a.H, h0 + f.q_heads);
    const int rows = min(f.span, ROWS), abreast = ROWS / rows;
    auto position_of = [&](int t) { return a.rot && t < w1 ? a.positions[t] : 0; };
    int position = position_of(w0 + r % rows);
    for (int t = w0 + r % rows; t < w1; t += rows) {
      const int next = position_of(t + rows);
      float c[8], s[8];
      bf16* dst = (bf16*)a.q_out + (size_t)t * a.q_stride;
      const bf16* src = (const bf16*)a.qkv + (size_t)t * row_elems;
      bool first = true;
      // two heads' rows on their way at a time, and the table's: no load can pass a store of unknown address by itself
      for (int h = h0 + r / rows; h < h1; h += HEADS * abreast) {
        uint4 u[HEADS], v[HEADS];
        if (!PART) {
#pragma unroll
          for (int k = 0; k < HEADS; ++k) {
            const int hk = min(h + k * abreast, h1 - 1);
            u[k] = *reinterpret_cast<const uint4*>(src + hk * D + 8 * j);
            v[k] = *reinterpret_cast<const uint4*>(src + hk * D + HALF + 8 * j);
          }
        }
        if (first && a.rot) load_table(a, position, HALF, j, c, s);
        first = false;
#pragma unroll
        for (int k = 0; k < HEADS; ++k) {
          const int hk = h + k * abreast;
          if (hk >= h1) break;
          float x[16];
          if (PART) load16<PART>(f, t, row_elems, hk * D + 8 * j, hk * D + HALF + 8 * j, x);
          else widen16(u[k], v[k], x);
          if (a.rot) turn(x, c, s);
          unsigned w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned*>(&p);
          }
          *reinterpret_cast<uint4*>(dst + hk * D + 8 * j) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4*>(dst + hk * D + HALF + 8 * j) = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
      position = next;
    }
    return;
  }
  const int kv = blockIdx.y / a.KVH, kvh = blockIdx.y % a.KVH, lane = tid & 31;
  __shared__ int slot_s[SPAN_MAX], lead_s[SPAN_MAX], edge_s[2], fresh_s[SPAN_MAX];
  __shared__ unsigned mask_s[2][2], amax_s[SPAN_MAX];             // leaders, live tokens
  __shared__ float inv_s[SPAN_MAX];
  const int col = (a.H + kv * a.KVH + kvh) * D + 8 * j;
  auto load_row = [&](int t, float (&x)[16]) {
    load16<PART>(f, t, row_elems, col, col + HALF, x);
    if (kv == 0 && a.rot) {
      float c[8], s[8];
      load_table(a, a.positions[t], HALF, j, c, s);
      turn(x, c, s);
    }
  };
  // All that the first trip to memory can bring: the span's slots, 128 slots to either side (its first and last run may go on there), and
  // the span's rows, if it is no more of them than the block takes in one turn.
  const bool back = tid < 32;
  int around[4];
  auto neighbour = [&](int t) { return t >= 0 && t < a.T ? max(a.slots[t], -1) : -2; };         // (-2: no token there; -1: one that is not written)
  if (tid < 64) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = back ? w0 - 1 - (u * 32 + lane) : w1 + u * 32 + lane;
      around[u] = neighbour(t);
    }
  }
  if (tid < SPAN_MAX) {
    const int t = w0 + tid;
    slot_s[tid] = t < w1 ? a.slots[t] : -1;
    fresh_s[tid] = 0;
    amax_s[tid] = 0;
  }
  float x[16];
  const bool short_span = f.span <= ROWS;
  if (short_span && w0 + r < w1) load_row(w0 + r, x);
  __syncthreads();
  if (tid < SPAN_MAX) {
    const unsigned m = __ballot_sync(0xffffffffu, slot_s[tid] >= 0);
    if (lane == 0) mask_s[1][tid >> 5] = m;
  }
  __syncthreads();
  const unsigned long long live = mask_s[1][0] | (unsigned long long)mask_s[1][1] << 32;
  if (tid < SPAN_MAX) {
    const unsigned long long below = live & ((1ull << tid) - 1);
    const int s = slot_s[tid], pg = s / a.page;
    const bool lead = s >= 0 && (below == 0 || slot_s[63 - __clzll((long long)below)] / a.page != pg);
    const unsigned m = __ballot_sync(0xffffffffu, lead);
    if (lane == 0) mask_s[0][tid >> 5] = m;
  }
  __syncthreads();
  const unsigned long long leads = mask_s[0][0] | (unsigned long long)mask_s[0][1] << 32;
  if (live == 0) return;
  const int n_runs = __popcll(leads);
  auto run_at = [&](int i) { return __popcll(leads & (~0ull >> (63 - i))) - 1; };
  // the scales that the runs' pages have: on their way while the rows' maxima are found
  float held = 0.f;
  if (tid < SPAN_MAX && (leads >> tid & 1)) {
    lead_s[run_at(tid)] = tid;
    held = a.scale[kv][(size_t)(slot_s[tid] / a.page) * a.KVH + kvh];
  }
  if (tid < 64) {
    // where the first run begins (warp 0) and the last one ends (warp 1): 128 tokens a turn
    const int pg = slot_s[back ? __ffsll((long long)live) - 1 : 63 - __clzll((long long)live)] / a.page;
    int edge = back ? w0 : w1, at = back ? w0 - 1 : w1;           // tokens [edge of the run]; next token to look at
    for (;;) {
      bool ended = false;
#pragma unroll
      for (int u = 0; u < 4 && !ended; ++u) {
        const unsigned other = __ballot_sync(0xffffffffu, around[u] == -2 || (around[u] >= 0 && around[u] / a.page != pg));
        unsigned same = __ballot_sync(0xffffffffu, around[u] >= 0 && around[u] / a.page == pg);
        if (other) same &= (other & (~other + 1)) - 1;            // only those before the first that is not of the run
        if (same) {
          const int far = u * 32 + 31 - __clz(same);
          edge = back ? at - far : at + far + 1;
        }
        ended = other != 0;
      }
      if (ended) break;
      at += back ? -128 : 128;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int t = back ? at - (u * 32 + lane) : at + u * 32 + lane;
        around[u] = neighbour(t);
      }
    }
    if (lane == 0) edge_s[back ? 0 : 1] = edge;
  }
  __syncthreads();
  const int e0 = edge_s[0], e1 = edge_s[1];
  auto slot_of = [&](int t) { return t >= w0 && t < w1 ? slot_s[t - w0] : a.slots[t]; };
  auto run_of = [&](int t) { return t < w0 ? 0 : (t >= w1 ? n_runs - 1 : run_at(t - w0)); };
  const bool own = short_span && e0 >= w0 && e1 <= w1;            // the runs lie in the span, whose rows are in registers
  for (int base = own ? w0 : e0; base < e1; base += ROWS) {       // (every lane of a warp takes every turn: the maxima are shuffled)
    const int t = base + r, s = t < e1 ? slot_of(t) : -1;
    unsigned amax = 0;
    if (s >= 0) {
      if (!own) load_row(t, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = max(amax, __float_as_uint(fabsf(x[i])));
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (s >= 0 && j == 0) {
      const int run = run_of(t);
      atomicMax(&amax_s[run], amax);
      if (s % a.page == 0) fresh_s[run] = 1;
    }
  }
  __syncthreads();
  // (a run belongs to the block that has its first token)
  auto begins_here = [&](int run) { return run > 0 || e0 >= w0; };
  __shared__ float held_s[SPAN_MAX], now_s[SPAN_MAX];
  if (tid < SPAN_MAX && (leads >> tid & 1)) {
    const int run = run_at(tid);
    const float need = scale_for(amax_s[run]), now = fresh_s[run] ? need : larger_scale(held, need);
    held_s[run] = held;
    now_s[run] = now;
    inv_s[run] = inverse_scale(now);
  }
  __syncthreads();
  auto page_rows = [&](int slot) { return a.cache[kv] + ((size_t)(slot / a.page) * a.KVH + kvh) * a.page * D; };
  for (int run = 0; run < n_runs; ++run) {
    if (fresh_s[run] || !(now_s[run] > held_s[run]) || !begins_here(run)) continue;         // (uniform over the block)
    unsigned char* rows = page_rows(slot_s[lead_s[run]]);
    const float ratio = held_s[run] * inv_s[run];
    const int first = w0 + lead_s[run], last = run + 1 < n_runs ? w0 + lead_s[run + 1] : e1;
    for (int row = r; row < a.page; row += ROWS) {
      bool written = false;
      for (int t = first; t < last; ++t) {
        const int s = slot_of(t);
        written = written || (s >= 0 && s % a.page == row);
      }
      if (written) continue;
      uint4* p = reinterpret_cast<uint4*>(rows + (size_t)row * D + 16 * j);
      uint4 v = *p;
      unsigned* w = reinterpret_cast<unsigned*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = four_e4m3(from_e4m3(w[i] & 255) * ratio, from_e4m3(w[i] >> 8 & 255) * ratio, from_e4m3(w[i] >> 16 & 255) * ratio,
                         from_e4m3(w[i] >> 24) * ratio);
      *p = v;
    }
  }
  for (int t = w0 + r; t < w1; t += ROWS) {
    const int s = slot_s[t - w0];
    if (s < 0) continue;
    if (!own) load_row(t, x);
    const float inv = inv_s[run_at(t - w0)];
    unsigned w[4] = {0, 0, 0, 0};
    if (inv != 0.f) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = four_e4m3(x[4 * i] * inv, x[4 * i + 1] * inv, x[4 * i + 2] * inv, x[4 * i + 3] * inv);
    }
    unsigned char* dst = page_rows(s) + (size_t)(s % a.page) * D + 8 * j;
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(dst + HALF) = make_uint2(w[2], w[3]);
  }
  if (tid < n_runs && begins_here(tid)) a.scale[kv][(size_t)(slot_s[lead_s[tid]] / a.page) * a.KVH + kvh] = now_s[tid];
}

template <int D, int THREADS>
cudaError_t launch_fast(FastArgs f, int span, cudaStream_t s) {
  const WriteArgs& a = f.w;
  constexpr int ROWS = THREADS / (D / 16);
  f.span = span;
  f.kv_blocks = a.cache[0] != nullptr ? 2 * a.KVH : 0;
  // query heads a block (they share a table row's conversion): as many as keep 4,096 lanes an SM, at least one row of lanes each (7,787 tokens, 2 / 4
  // / 7 / 14 heads 31 / 31 / 36 / 43 us)
  const int least = f.span < ROWS ? ROWS / f.span : 1;
  const long long lanes = (long long)a.T * (D / 16) * a.H, want = lanes / ((long long)ts_sm_count() * 4096);
  f.q_heads = (int)(want < least ? least : (want > a.H ? a.H : want));
  const dim3 grid(ceil_div(a.T, f.span), f.kv_blocks + ceil_div(a.H, f.q_heads)), block(THREADS);
  return f.part != nullptr ? ts_launch(kv_write_q8_fast_kernel<D, THREADS, true>, grid, block, 0, s, f)
                           : ts_launch(kv_write_q8_fast_kernel<D, THREADS, false>, grid, block, 0, s, f);
}
// Threads a block and tokens a block.  Every block of a page's rows reads all of them, in turns of as many rows as its threads hold: of 256 threads
// it takes half as long (us at 128 / 256, spans of 16: a portion of 200 tokens, 28 heads over 4, 12.6 / 8.6, of 700 14.1 / 9.8; 64 single
// tokens in pages of 16 5.2 / 5.0), and wider spans read them in fewer blocks (256 threads, spans of 16 / 32 / 64: 1,999 tokens 19.2 / 14.7
// / 13.6, 1,000 10.5 / 10.5 / 10.9; 64 single tokens 5.0 / 6.2 / 10.8).  Where the work is many times what the chip holds smaller blocks fill it better.
// Spans of 64, 128 / 256 threads, pages of 64:
//   tokens                 1,500          2,500          4,096          5,500          7,787          8,192
//   14 over 2 of 64      9.0 /  7.6     9.7 /  7.9    11.7 /  9.0    12.1 / 10.9    13.5 / 14.9    13.7 / 15.5
//   12 over 2 of 128    14.8 / 10.0    17.0 / 10.9    20.3 / 13.3    20.6 / 15.8    21.8 / 20.8    21.9 / 21.8
//   28 over 4           19.1 / 12.4    20.5 / 15.7    22.0 / 23.6    24.1 / 26.7    31.8 / 37.1    35.3 / 40.0
//   40 over 8           20.1 / 15.4    22.1 / 24.3    29.1 / 33.1    38.8 / 43.5    53.3 / 60.4    55.2 / 62.5
// The border, 4,096 tokens for every model, is a compromise: of few heads it comes too early (12 over 2 of 4,097 tokens get 20.2 where 13.3 is
// had), of many too late (40 over 8 of 2,500 and 4,096 tokens lose 2 and 4 us).  A few tokens want a block each (8 single tokens, 128 threads, spans
// of 1 / 16: 3.8 / 4.2).
template <int D>
cudaError_t launch_fast(const FastArgs& f, cudaStream_t s) {
  const int T = f.w.T;
  if (T <= 8) return launch_fast<D, 128>(f, 1, s);
  if (T <= 4096) return launch_fast<D, 256>(f, T <= 1024 ? 16 : SPAN_MAX, s);
  return launch_fast<D, 128>(f, SPAN_MAX, s);
}

}  // namespace

static bool write_is_fast(int D, int rot, int dtype) { return dtype == TS_BF16 && (D == 64 || D == 128) && (rot == 0 || rot == D); }

// Whether the write also takes an unfinished product (its partial sums).
TS_API int ts_rope_kv_write_q8_takes_parts(int D, int rot, int dtype) { return write_is_fast(D, rot, dtype); }

// qkv [T, (H + 2 KVH) * D], q_out [T, H * D] with rows q_stride elements apart.  k_cache null: queries only.  part (float
// [splits, T, (H + 2 KVH) * D]) set: qkv is the sum of the splits and the bias, rounded, and is not read.
// The arguments come as one record (as do those of the other entry points of this cache: converting twenty of them one by one costs
// the caller 2 us a call, a fifth of what a decode step's write takes it).
struct WriteCall {
  void* q_out;
  const void* qkv;
  const int* positions;
  const float *cos_t, *sin_t;
  void *k_cache, *v_cache;
  float *k_scale, *v_scale;
  const int* slots;
  const float* part;
  const void* bias;
  long long q_stride;
  int T, H, KVH, D, rot, page, dtype, splits;
};

TS_API int ts_rope_kv_write_q8_record() { return (int)sizeof(WriteCall); }

TS_API int ts_rope_kv_write_q8(const void* record, void* stream) {
  const WriteCall& c = *(const WriteCall*)record;
  void *const q_out = c.q_out, *const k_cache = c.k_cache, *const v_cache = c.v_cache;
  const void *const qkv = c.qkv, *const bias = c.bias;
  const int *const positions = c.positions, *const slots = c.slots;
  const float *const cos_t = c.cos_t, *const sin_t = c.sin_t, *const part = c.part;
  float *const k_scale = c.k_scale, *const v_scale = c.v_scale;
  const long long q_stride = c.q_stride;
  const int T = c.T, H = c.H, KVH = c.KVH, D = c.D, rot = c.rot, page = c.page, dtype = c.dtype, splits = c.splits;
  if (T <= 0) return 0;
  if (H <= 0 || KVH <= 0 || D <= 0 || page <= 0 || H + 2 * KVH > 65535)
    TS_REFUSE(TS_ERR_SHAPE, "ts_rope_kv_write_q8: H=%d KVH=%d D=%d page=%d", H, KVH, D, page);
  if (rot < 0 || rot > D || (rot & 1)) TS_REFUSE(TS_ERR_SHAPE, "ts_rope_kv_write_q8: rotary_dim %d for head_dim %d", rot, D);
  if (rot > 0 && (cos_t == nullptr || sin_t == nullptr)) TS_REFUSE(TS_ERR_SHAPE, "ts_rope_kv_write_q8: tables missing");
  if (k_cache != nullptr && (v_cache == nullptr || k_scale == nullptr || v_scale == nullptr || slots == nullptr))
    TS_REFUSE(TS_ERR_SHAPE, "ts_rope_kv_write_q8: keys without values, scales or slots");
  if (dtype != TS_F32 && dtype != TS_BF16) TS_REFUSE(TS_ERR_DTYPE, "ts_rope_kv_write_q8: dtype %d", dtype);
  // (turned queries over keys or halves that others still read)
  const size_t elem = dtype == TS_F32 ? 4 : 2;
  const char *const q0 = (const char*)q_out, *const q1 = q0 + ((size_t)(T - 1) * q_stride + (size_t)H * D) * elem;
  if (q_stride < 0 || (q0 < (const char*)qkv + (size_t)T * (H + 2 * KVH) * D * elem && (const char*)qkv < q1))
    TS_REFUSE(TS_ERR_SHAPE, "ts_rope_kv_write_q8: the queries' rows lie in qkv");
  WriteArgs a = {qkv, q_out, q_stride, positions, cos_t, sin_t, {(unsigned char*)k_cache, (unsigned char*)v_cache},
                 {k_scale, v_scale}, slots, T, H, KVH, D, rot, page};
  cudaStream_t s = (cudaStream_t)stream;
  const bool aligned = (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)k_cache | (uintptr_t)v_cache |
                         (uintptr_t)part) & 15) == 0 && q_stride % 8 == 0;
  if (write_is_fast(D, rot, dtype) && aligned) {
    FastArgs f = {a, part, (const bf16*)bias, splits, 0, 0, 0};
    const cudaError_t e = D == 64 ? launch_fast<64>(f, s) : launch_fast<128>(f, s);
    if (e != cudaSuccess) TS_REFUSE((int)e, "ts_rope_kv_write_q8: %s", cudaGetErrorString(e));
    TS_LAUNCH_CHECK();
  }
  if (part != nullptr) TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_rope_kv_write_q8: partial sums with head_dim %d, rotary_dim %d or buffers that "
                                 "are not on 16 bytes", D, rot);
  const dim3 grid(T, k_cache != nullptr ? H + 2 * KVH : H), block(D >= 128 ? 128 : 64);
  if (dtype == TS_F32) ts_launch(kv_write_q8_kernel<float>, grid, block, 0, s, a);
  else ts_launch(kv_write_q8_kernel<bf16>, grid, block, 0, s, a);
  TS_LAUNCH_CHECK();
}
