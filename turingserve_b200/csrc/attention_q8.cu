// Paged grouped-query attention over an 8-bit cache (q8_cache.cuh), any sizes, 32-bit arithmetic: the float32 path and the
// shapes that the tensor-core kernels do not take.
//
// Same semantics as attention_generic.cu: query token t of a request at position p = seq_len - q_len + t sees keys j <= p,
// with a window w only j > p - w; query head h reads kv head h / G; a request with seq_len 0 gives zeros.  Keys and values
// are e4m3 times their page's scale.  Rows that see a page whose scale is NaN give NaN, and only those: the tile's key rows
// carry the NaN (masked scores are dropped by selection), its value rows are zeros then (zero weights would keep a NaN).
//
// Work split: one block per (16 rows, kv head, request), a row one (token, head-in-group) pair; 32 keys a turn, a lane
// scores one, then each lane accumulates its share of the head's columns.
#include "q8_cache.cuh"

namespace {

constexpr int ROWS = 16, KT = 32, NWARPS = 4, RPW = ROWS / NWARPS, MAX_DPL = 8;

template <typename T>
__global__ void __launch_bounds__(NWARPS * 32)
attention_q8_kernel(T* __restrict__ out, long long o_ts, const T* __restrict__ q, long long q_ts,
                    const unsigned char* __restrict__ k_cache, const unsigned char* __restrict__ v_cache,
                    const float* __restrict__ k_scale, const float* __restrict__ v_scale, const int* __restrict__ block_tables,
                    const int* __restrict__ q_start, const int* __restrict__ seq_lens, int table_width, int H, int KVH, int D,
                    int page, float scale, int window) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ float smem[];
  const int b = blockIdx.z, kvh = blockIdx.y, G = H / KVH;
  const int qs = q_start[b], q_len = q_start[b + 1] - qs, seq_len = seq_lens[b];
  const int row0 = blockIdx.x * ROWS, n_rows = q_len * G;
  if (row0 >= n_rows) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int dpl = (D + 31) / 32, prefix = seq_len - q_len;

  float* q_s = smem;                         // [ROWS][D]
  float* k_s = q_s + ROWS * D;               // [KT][D + 1]
  float* v_s = k_s + KT * (D + 1);           // [KT][D]
  __shared__ size_t key_off[KT];
  __shared__ float key_scale[KT], val_scale[KT];

  for (int idx = threadIdx.x; idx < ROWS * D; idx += blockDim.x) {
    const int row = row0 + idx / D, d = idx % D;
    q_s[idx] = row < n_rows ? to_f(q[(size_t)(qs + row / G) * q_ts + (size_t)(kvh * G + row % G) * D + d]) : 0.f;
  }
  const int last_row = min(row0 + ROWS, n_rows) - 1;
  const int j_hi = prefix + last_row / G;                           // last key any row of the block sees
  const int j_lo = window > 0 ? max(0, prefix + row0 / G - window + 1) : 0;

  float m[RPW], l[RPW], acc[RPW][MAX_DPL];
  int p_row[RPW], lo_row[RPW];
#pragma unroll
  for (int r = 0; r < RPW; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < MAX_DPL; ++i) acc[r][i] = 0.f;
    const int row = row0 + warp * RPW + r;
    p_row[r] = row < n_rows ? prefix + row / G : -1;
    lo_row[r] = window > 0 ? max(0, p_row[r] - window + 1) : 0;
  }

  if (seq_len > 0)
    for (int j0 = j_lo; j0 <= j_hi; j0 += KT) {
      __syncthreads();
      if (threadIdx.x < KT) {
        const int j = j0 + threadIdx.x, lp = j / page;
        const int pg = (j <= j_hi && lp < table_width) ? block_tables[(size_t)b * table_width + lp] : -1;
        float ks = 0.f, vs = 0.f;
        if (pg >= 0) {
          ks = k_scale[(size_t)pg * KVH + kvh];
          vs = v_scale[(size_t)pg * KVH + kvh];
          if (vs != vs) {
            ks = vs;
            vs = 0.f;
          }
        }
        key_off[threadIdx.x] = pg >= 0 ? (((size_t)pg * KVH + kvh) * page + (size_t)(j % page)) * D : (size_t)-1;
        key_scale[threadIdx.x] = ks;
        val_scale[threadIdx.x] = vs;
      }
      __syncthreads();
      for (int idx = threadIdx.x; idx < KT * D; idx += blockDim.x) {
        const int kk = idx / D, d = idx % D;
        const size_t off = key_off[kk];
        const bool there = off != (size_t)-1;
        k_s[kk * (D + 1) + d] = there ? q8::from_e4m3(k_cache[off + d]) * key_scale[kk] : 0.f;
        v_s[kk * D + d] = there ? q8::from_e4m3(v_cache[off + d]) * val_scale[kk] : 0.f;
      }
      __syncthreads();
      const int j = j0 + lane;
#pragma unroll
      for (int r = 0; r < RPW; ++r) {
        if (p_row[r] < j0) continue;                 // the whole turn lies in this row's future (warp-uniform)
        const float* qr = q_s + (warp * RPW + r) * D;
        const float* kr = k_s + lane * (D + 1);
        float s = 0.f;
        for (int d = 0; d < D; ++d) s = fmaf(qr[d], kr[d], s);
        const bool ok = j <= p_row[r] && j >= lo_row[r];
        s = ok ? s * scale : -INFINITY;
        const float m_new = fmaxf(m[r], warp_max(s));
        const float ref = m_new == -INFINITY ? 0.f : m_new;          // (a NaN is no maximum: it shows in the exponential)
        const float p = ok ? expf(s - ref) : 0.f;
        const float corr = m[r] == -INFINITY ? (l[r] != l[r] ? 1.f : 0.f) : expf(m[r] - ref);
        l[r] = l[r] * corr + warp_sum(p);
        m[r] = m_new;
#pragma unroll
        for (int i = 0; i < MAX_DPL; ++i) acc[r][i] *= corr;
        for (int kk = 0; kk < KT; ++kk) {
          const float pk = __shfl_sync(0xffffffffu, p, kk);
          const float* vr = v_s + kk * D;
#pragma unroll
          for (int i = 0; i < MAX_DPL; ++i) {
            const int d = lane + 32 * i;
            if (i < dpl && d < D) acc[r][i] = fmaf(pk, vr[d], acc[r][i]);
          }
        }
      }
    }

#pragma unroll
  for (int r = 0; r < RPW; ++r) {
    const int row = row0 + warp * RPW + r;
    if (row >= n_rows) continue;
    const float inv = l[r] > 0.f ? 1.f / l[r] : l[r];                // nothing seen: 0; NaN stays
    T* o = out + (size_t)(qs + row / G) * o_ts + (size_t)(kvh * G + row % G) * D;
#pragma unroll
    for (int i = 0; i < MAX_DPL; ++i) {
      const int d = lane + 32 * i;
      if (i < dpl && d < D) o[d] = from_f<T>(acc[r][i] * inv);
    }
  }
}

template <typename T>
int launch(const q8::AttendCall& c, cudaStream_t s) {
  const int D = c.D;
  const size_t smem = sizeof(float) * ((size_t)ROWS * D + (size_t)KT * (D + 1) + (size_t)KT * D);
  static size_t configured = 0;
  if (smem > 48 * 1024 && smem > configured) {
    cudaError_t e = cudaFuncSetAttribute(attention_q8_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) TS_REFUSE((int)e, "ts_attention_q8: shared memory %zu: %s", smem, cudaGetErrorString(e));
    configured = smem;
  }
  const long long tiles = ((long long)c.max_q_len * (c.H / c.KVH) + ROWS - 1) / ROWS;
  if (tiles > 0x7fffffffLL) TS_REFUSE(TS_ERR_LIMIT, "ts_attention_q8: portions of %d tokens", c.max_q_len);
  ts_launch(attention_q8_kernel<T>, dim3((unsigned)tiles, c.KVH, c.B), dim3(NWARPS * 32), smem, s, (T*)c.out, c.o_ts, (const T*)c.q, c.q_ts,
            (const unsigned char*)c.k_cache, (const unsigned char*)c.v_cache, c.k_scale, c.v_scale, c.block_tables, c.q_start, c.seq_lens,
            c.table_width, c.H, c.KVH, D, c.page, c.scale, c.window);
  TS_LAUNCH_CHECK();
}

}  // namespace

// q, out: rows [H, D] o_ts / q_ts elements apart.  window <= 0: none.
TS_API int ts_attention_q8_record() { return (int)sizeof(q8::AttendCall); }

TS_API int ts_attention_q8(const void* record, void* stream) {
  const q8::AttendCall& c = *(const q8::AttendCall*)record;
  const int B = c.B, max_q_len = c.max_q_len, H = c.H, KVH = c.KVH, D = c.D, page = c.page, dtype = c.dtype;
  if (B <= 0 || max_q_len <= 0) return 0;
  if (KVH <= 0 || H % KVH || page <= 0) TS_REFUSE(TS_ERR_SHAPE, "ts_attention_q8: %d heads over %d kv heads, pages of %d", H, KVH, page);
  if (D <= 0 || D > 32 * MAX_DPL) TS_REFUSE(TS_ERR_LIMIT, "ts_attention_q8: head_dim %d (limit %d)", D, 32 * MAX_DPL);
  if (B > 65535 || KVH > 65535) TS_REFUSE(TS_ERR_LIMIT, "ts_attention_q8: %d requests / %d kv heads per launch", B, KVH);
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == TS_F32)
    return launch<float>(c, s);
  if (dtype == TS_BF16)
    return launch<bf16>(c, s);
  TS_REFUSE(TS_ERR_DTYPE, "ts_attention_q8: dtype %d", dtype);
}
