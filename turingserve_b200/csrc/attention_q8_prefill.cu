// Attention of prompt portions over an 8-bit paged cache (q8_cache.cuh) on the 5th-generation tensor cores: bfloat16 queries, heads
// of 64 or 128, pages of a multiple of 16 tokens, any group size.
//
// Mathematics as in attention_q8_decode.cu: weights P = 2^(t - M), t = score + log2 of the value's scale, on values as they lie in
// the pages; the denominator sums P / scale.  Both products take half floats: keys and values as they are (e4m3 fits whole), queries
// scaled by a power of two a row, P below 2^8.  The scales are constants of 16 keys, so a score costs one fused multiply-add as it would
// without them, and a sum one more for 16 weights.
//
// One block = NR tiles of 128 query rows (a row is a (token, head-in-group) pair of one kv head) over the same keys, 64 a turn.
// Softmax warps: eight a row tile, row r = tensor-memory lane r belongs to two threads, each half of a turn's keys; they exchange their
// maxima through shared memory once a turn.  One warp issues the products (one lane): S(t) = Q K(t)^T into one of two buffers, two
// turns ahead; O += P(t) V(t), P read from tensor memory where it lies over its own scores.  Four warps turn the pages' bytes into
// half floats, two the keys and two the values: 16 bytes a load, a turn's loads in flight while the turn before is converted, stored with
// the 128-byte swizzle that the products read (values with keys along the rows: MN-major).  Rows outside the visible range are zeros.
// With NR = 2 a converted tile serves 256 rows: the conversion is half as much work beside each row's exponentials, and one block fills
// an SM; NR = 1 is for launches of few row tiles, which are as slow as their longest block.
// The reference M moves only when a row's maximum has grown by more than 2^8 since: then O is rescaled in tensor memory.  Every wait is
// bounded; a block that gives up records where, stops, and frees its tensor memory.
//
// NaN: a page whose scale is NaN (either) gives NaN scores, which the rows that do not see it drop by selection; its values are
// finite bytes (writes store zeros under such a scale), so zero weights stay zeros.
#include "q8_cache.cuh"
#include "tc_utils.cuh"

namespace {

using namespace tc;

constexpr int TQ = 128, TK = 64, STAGES = 2, SCALE_STAGES = 4, CONV_WARPS = 4;
constexpr float RESCALE_STEP = 8.f;
constexpr float LOG2E_P = 1.4426950408889634f;

template <int HD, int NR>
struct Shape {
  static constexpr int SOFT_WARPS = 8 * NR, MMA_WARP = SOFT_WARPS, CONV_WARP = MMA_WARP + 1;
  static constexpr int THREADS = (SOFT_WARPS + 1 + CONV_WARPS) * 32;
  static constexpr uint32_t Q_BYTES = TQ * HD * 2, KV_BYTES = TK * HD * 2, HALF_Q = TQ * 128, HALF_K = TK * 128;
  static constexpr uint32_t ROW_COLS = 2 * TK + HD;                // tensor-memory columns of a row tile: two score buffers, O
  static constexpr uint32_t TMEM_COLS = ROW_COLS * NR <= 256 ? 256 : 512;
  // behind the tiles: barriers, the tensor memory's address, the abort flag, maxima [NR][2][128], scales [4][4] float4
  static constexpr int BARS = 4 * STAGES + NR * (2 + 2 + 1 + 1 + 4 + 4);
  static constexpr size_t TILES = NR * Q_BYTES + 2 * STAGES * KV_BYTES;
  static constexpr size_t SMEM = TILES + BARS * 8 + 16 + NR * 2 * TQ * 4 + SCALE_STAGES * 4 * 16 + 16;
};

struct PreArgs {
  bf16* out;
  long long o_ts;
  const bf16* q;
  long long q_ts;
  const unsigned char* cache[2];
  const float* scales[2];
  const int* block_tables;
  const int* q_start;
  const int* seq_lens;
  int table_width, H, KVH, page;
  float scale;
  int window;
  int* status;
};

// Instruction descriptor: half x half -> float, M = 128, N = n; A K-major, B K-major or (b_mn) MN-major.
__host__ __device__ constexpr uint32_t instr_half(int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

template <int HD, int NR>
__global__ void __launch_bounds__(Shape<HD, NR>::THREADS, 1) attention_q8_prefill_kernel(const PreArgs a) {
  using SH = Shape<HD, NR>;
  constexpr uint32_t KV_BYTES = SH::KV_BYTES, HALF_K = SH::HALF_K, HALF_Q = SH::HALF_Q, ROW_COLS = SH::ROW_COLS, O_COL = 2 * TK;
  constexpr int HC = HD / 2, ROWS = NR * TQ, KT = TK / 2;
  pdl_launch_dependents();
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* q_s = smem;                                       // [NR][HD / 64][128][128 B]
  unsigned char* k_s = q_s + NR * SH::Q_BYTES;                     // [STAGES][HD / 64][64][128 B]
  unsigned char* v_s = k_s + STAGES * KV_BYTES;
  uint64_t* full_k = reinterpret_cast<uint64_t*>(v_s + STAGES * KV_BYTES);
  uint64_t* empty_k = full_k + STAGES;
  uint64_t* full_v = empty_k + STAGES;
  uint64_t* empty_v = full_v + STAGES;
  uint64_t* bar_s = empty_v + STAGES;                              // [NR][2]: that score buffer is complete
  uint64_t* bar_p = bar_s + 2 * NR;                                // [NR][2]: all rows have read S(t) and written P(t)
  uint64_t* bar_pv = bar_p + 2 * NR;                               // [NR]: an O product is complete
  uint64_t* bar_o = bar_pv + NR;                                   // [NR]: the last one
  uint64_t* bar_x = bar_o + NR;                                    // [NR][4]: both threads of the rows have left their maxima
  uint64_t* bar_r = bar_x + 4 * NR;                                // [NR][4]: both have read the other's
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_r + 4 * NR);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* max_x = reinterpret_cast<float*>(tmem_slot + 4);          // [NR][2][128]
  float4* scale_s = reinterpret_cast<float4*>(smem + ((SH::TILES + SH::BARS * 8 + 16 + NR * 2 * TQ * 4 + 15) & ~(size_t)15));

  const int b = blockIdx.z, kvh = blockIdx.y, G = a.H / a.KVH;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();                                                      // what it reads is written by kernels before
  const int qs = a.q_start[b], q_len = a.q_start[b + 1] - qs, seq_len = a.seq_lens[b];
  const int n_rows = q_len * G, n_blocks = (n_rows + ROWS - 1) / ROWS;
  if ((int)blockIdx.x >= n_blocks) return;
  const int row0 = (n_blocks - 1 - blockIdx.x) * ROWS;             // longest blocks first
  const int prefix = seq_len - q_len;

  if ((smem_u32(smem) & 1023u) != 0) {                             // the swizzled tiles need 1024-byte alignment
    if (tid == 0) atomicCAS(a.status, 0, 29);
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_k[s], CONV_WARPS / 2);
      mbar_init(&empty_k[s], 1);
      mbar_init(&full_v[s], CONV_WARPS / 2);
      mbar_init(&empty_v[s], 1);
    }
    for (int r = 0; r < NR; ++r) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bar_s[2 * r + i], 2);                           // the product's end, and the issuing thread, which saw the scales
        mbar_init(&bar_p[2 * r + i], 2 * TQ);
      }
      mbar_init(&bar_pv[r], 1);
      mbar_init(&bar_o[r], 1);
      for (int i = 0; i < 4; ++i) {
        mbar_init(&bar_x[4 * r + i], 64);
        mbar_init(&bar_r[4 * r + i], 64);
      }
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == SH::MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(SH::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  const int last_row = min(row0 + ROWS, n_rows) - 1;
  const int j_hi = prefix + last_row / G;                          // the last key that any row sees, and the first
  const int key_lo = a.window > 0 ? max(0, prefix + row0 / G - a.window + 1) : 0;
  const int j_lo = key_lo & ~15;
  const int n_tiles = (seq_len > 0 && j_hi >= key_lo) ? (j_hi - j_lo) / TK + 1 : 0;

  // a softmax thread's row tile, row, and which half of a turn's keys (and of the head's columns) it takes
  const int rt = warp >> 3, lane_row = tid & (TQ - 1), hh = (warp >> 2) & 1;
  const bool softmax = warp < SH::SOFT_WARPS;
  const int row = row0 + rt * TQ + lane_row;
  const bool row_ok = softmax && row < n_rows;
  const int tok = row_ok ? row / G : 0, g = row_ok ? row % G : 0;
  const int pos = row_ok ? prefix + tok : -1;

  // Q rows -> shared memory as half floats, K-major with the 128-byte swizzle (16-byte piece c of row r at c ^ (r & 7))
  float factor = 0.f;
  uint4 qv[HC / 8];
  if (softmax) {
    const bf16* src = a.q + (size_t)(qs + tok) * a.q_ts + (size_t)(kvh * G + g) * HD + hh * HC;
    float amax = 0.f;
#pragma unroll
    for (int cc = 0; cc < HC / 8; ++cc) {
      qv[cc] = row_ok ? *reinterpret_cast<const uint4*>(src + cc * 8) : make_uint4(0u, 0u, 0u, 0u);
      const unsigned w[4] = {qv[cc].x, qv[cc].y, qv[cc].z, qv[cc].w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        amax = fmaxf(amax, fmaxf(q8::abs_or_inf(__uint_as_float(w[i] << 16)), q8::abs_or_inf(__uint_as_float(w[i] & 0xffff0000u))));
    }
    max_x[(rt * 2 + hh) * TQ + lane_row] = amax;
  }
  __syncthreads();
  if (softmax) {
    const float amax = fmaxf(max_x[rt * 2 * TQ + lane_row], max_x[(rt * 2 + 1) * TQ + lane_row]);
    const float to_half = q8::query_to_half(amax, a.scale * LOG2E_P, factor);
#pragma unroll
    for (int cc = 0; cc < HC / 8; ++cc) {
      const unsigned w[4] = {qv[cc].x, qv[cc].y, qv[cc].z, qv[cc].w};
      unsigned h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        h[i] = q8::pack_half(__uint_as_float(w[i] << 16) * to_half, __uint_as_float(w[i] & 0xffff0000u) * to_half);
      const int c = hh * (HC / 8) + cc;
      *reinterpret_cast<uint4*>(q_s + rt * SH::Q_BYTES + (c >> 3) * HALF_Q + lane_row * 128 + (((c & 7) ^ (lane_row & 7)) << 4)) =
          make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= SH::CONV_WARP) {
    // ================= converters: warps 0 and 1 the keys (and the scales), 2 and 3 the values =================
    constexpr int CPR = HD / 16, NP = TK * CPR / 64;               // 16-byte pieces of a row; pieces a thread takes of a tile
    constexpr int RPP = 64 / CPR;                                  // rows a turn of 64 threads covers
    const bool keys = warp < SH::CONV_WARP + 2;
    const int ct = (tid - SH::CONV_WARP * 32) & 63, c16 = ct % CPR, r0 = ct / CPR;
    const unsigned char* cache = keys ? a.cache[0] : a.cache[1];
    const int* table = a.block_tables + (size_t)b * a.table_width;
    // the page of 16 keys (lane & 3) of tile t, -1 outside; fetched two tiles ahead, for lanes 0 to 3's sake by all of them
    auto page_of = [&](int t) {
      const int j = j_lo + t * TK + (lane & 3) * 16, lp = j / a.page;
      return (t < n_tiles && j <= j_hi && lp < a.table_width) ? table[lp] : -1;
    };
    uint4 piece[NP];
    float ks = 0.f, vs = 0.f;
    auto load_scales = [&](int pg) {
      const size_t at = (size_t)max(pg, 0) * a.KVH + kvh;
      ks = pg >= 0 ? a.scales[0][at] : 0.f;
      vs = pg >= 0 ? a.scales[1][at] : 1.f;
    };
    auto load = [&](int t, int pg, int in_page, int i) {
      const int r = r0 + i * RPP, grp = r >> 4, j = j_lo + t * TK + r;
      const int p = __shfl_sync(0xffffffffu, pg, grp), in = __shfl_sync(0xffffffffu, in_page, grp);
      const bool there = p >= 0 && j >= key_lo && j <= j_hi;
      const unsigned char* src = cache + (((size_t)max(p, 0) * a.KVH + kvh) * a.page + in + (r & 15)) * HD + c16 * 16;
      piece[i] = there ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0u, 0u, 0u, 0u);
    };
    auto in_page_of = [&](int t) { return (j_lo + t * TK + (lane & 3) * 16) % a.page; };
    int pg_next = page_of(1);
    if (n_tiles > 0) {
      const int pg = page_of(0), in_page = in_page_of(0);
#pragma unroll
      for (int i = 0; i < NP; ++i) load(0, pg, in_page, i);
      if (keys) load_scales(pg);
    }
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      const int st = t % STAGES;
      if (t >= STAGES) {
        ok = mbar_wait(keys ? &empty_k[st] : &empty_v[st], (uint32_t)((t / STAGES - 1) & 1), a.status, keys ? 24 : 27, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      unsigned char* tile = (keys ? k_s : v_s) + st * KV_BYTES;
      if (keys && warp == SH::CONV_WARP && lane < 4)
        // (score factor, log2 of the value's scale, its inverse) of 16 keys
        scale_s[(t % SCALE_STAGES) * 4 + lane] = make_float4(vs != vs ? vs : ks, (float)((int)(__float_as_uint(vs) >> 23) - 127),
                                                             q8::inverse_scale(vs), 0.f);
      const int pg = pg_next, in_page = in_page_of(t + 1);
      pg_next = page_of(t + 2);
      if (keys) load_scales(pg);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = r0 + i * RPP, odd = c16 >> 2 & (HD == 128 ? 1 : 0);
        uint4 lo, hi;
        q8::halves_of(piece[i].x, lo.x, lo.y);
        q8::halves_of(piece[i].y, lo.z, lo.w);
        q8::halves_of(piece[i].z, hi.x, hi.y);
        q8::halves_of(piece[i].w, hi.z, hi.w);
        load(t + 1, pg, in_page, i);                               // (nothing behind the last tile: its pages are -1)
        // columns 16 c16 .. of the row: half c16 / 4 of the head, pieces 2 (c16 & 3) and the next; the second half's lanes begin with
        // the second piece, so that a row's eight lanes write to eight different places of a line
        unsigned char* line = tile + (c16 >> 2) * HALF_K + r * 128;
        const int first = 2 * (c16 & 3);
        *reinterpret_cast<uint4*>(line + (((first + odd) ^ (r & 7)) << 4)) = odd ? hi : lo;
        *reinterpret_cast<uint4*>(line + (((first + 1 - odd) ^ (r & 7)) << 4)) = odd ? lo : hi;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(keys ? &full_k[st] : &full_v[st]);
    }
  } else if (warp == SH::MMA_WARP) {
    // ================= product issue, one lane =================
    if (lane == 0 && n_tiles > 0) {
      auto issue_s = [&](int r, int t) {
        constexpr uint32_t idesc = instr_half(TK, false);
        const uint32_t qa = smem_u32(q_s + r * SH::Q_BYTES), ka = smem_u32(k_s + (t % STAGES) * KV_BYTES);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
          umma(tmem + r * ROW_COLS + (t & 1) * TK, smem_desc(qa + (ks >> 2) * HALF_Q + (ks & 3) * 32),
               smem_desc(ka + (ks >> 2) * HALF_K + (ks & 3) * 32), idesc, ks > 0 ? 1u : 0u);
        umma_commit(&bar_s[2 * r + (t & 1)]);
        mbar_arrive(&bar_s[2 * r + (t & 1)]);
        if (r == NR - 1) umma_commit(&empty_k[t % STAGES]);
      };
      auto issue_o = [&](int r, int t) {
        constexpr uint32_t idesc = instr_half(HD, true);
        const uint32_t va = smem_u32(v_s + (t % STAGES) * KV_BYTES), d = tmem + r * ROW_COLS + O_COL;
#pragma unroll
        for (int kk = 0; kk < TK / 16; ++kk)
          umma_ts(d, tmem + r * ROW_COLS + (t & 1) * TK + kk * 8, smem_desc_mn(va + kk * 16 * 128, HALF_K), idesc, (t > 0 || kk > 0) ? 1u : 0u);
        if (r == NR - 1) umma_commit(&empty_v[t % STAGES]);
        umma_commit(&bar_pv[r]);
        if (t + 1 == n_tiles) umma_commit(&bar_o[r]);
      };
      bool ok = true;
      for (int t = 0; t < 2 && t < n_tiles && ok; ++t) {
        ok = mbar_wait(&full_k[t], 0, a.status, 21, abort_flag);
        if (!ok) break;
        tc_fence_after();
        for (int r = 0; r < NR; ++r) issue_s(r, t);
      }
      for (int t = 0; t < n_tiles && ok; ++t)
        for (int r = 0; r < NR && ok; ++r) {
          ok = mbar_wait_spin(&bar_p[2 * r + (t & 1)], (uint32_t)((t >> 1) & 1), a.status, 26, abort_flag);
          if (ok && r == 0) ok = mbar_wait(&full_v[t % STAGES], (uint32_t)((t / STAGES) & 1), a.status, 23, abort_flag);
          if (!ok) break;
          tc_fence_after();
          issue_o(r, t);
          if (t + 2 < n_tiles) {
            if (r == 0) ok = mbar_wait(&full_k[t % STAGES], (uint32_t)(((t + 2) / STAGES) & 1), a.status, 28, abort_flag);
            if (!ok) break;
            tc_fence_after();
            issue_s(r, t + 2);                                     // over P(t), behind the product that reads it
          }
        }
    }
  } else {
    // ================= softmax: two threads per row = tensor-memory lane =================
    float m_ref = -INFINITY, l_run = 0.f;
    const int pair = warp & 3;                                     // warps `pair` and `pair + 4` of the row tile share 32 rows
    const uint32_t lane_addr = tmem + ((uint32_t)(pair * 32) << 16) + rt * ROW_COLS;
    uint64_t* const my_x = &bar_x[4 * rt + pair];
    uint64_t* const my_r = &bar_r[4 * rt + pair];
    float* const max_mine = max_x + (rt * 2 + hh) * TQ + lane_row;
    const float* const max_other = max_x + (rt * 2 + (hh ^ 1)) * TQ + lane_row;
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      const uint32_t s_addr = lane_addr + (t & 1) * TK;
      ok = mbar_wait_spin(&bar_s[2 * rt + (t & 1)], (uint32_t)((t >> 1) & 1), a.status, 22, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const int j0 = j_lo + t * TK + hh * KT;                      // this thread's first key of the turn
      uint32_t sv[KT];
      tmem_ld32(s_addr + hh * KT, sv);
      const float4 sc0 = scale_s[(t % SCALE_STAGES) * 4 + 2 * hh], sc1 = scale_s[(t % SCALE_STAGES) * 4 + 2 * hh + 1];
      const float f0 = sc0.x * factor, f1 = sc1.x * factor;
      tmem_wait_ld();
      float mx = -INFINITY;
      const bool all_visible = __all_sync(0xffffffffu, (j0 + KT - 1 <= pos) && (a.window <= 0 || j0 > pos - a.window));
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        float v = i < 16 ? fmaf(__uint_as_float(sv[i]), f0, sc0.y) : fmaf(__uint_as_float(sv[i]), f1, sc1.y);
        if (!all_visible) v = (j0 + i <= pos && (a.window <= 0 || j0 + i > pos - a.window)) ? v : -INFINITY;
        sv[i] = __float_as_uint(v);
        mx = fmaxf(mx, v);
      }
      if (t > 0) {
        ok = mbar_wait_spin(my_r, (uint32_t)((t - 1) & 1), a.status, 31, abort_flag);      // the last one has been read
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      *max_mine = mx;
      mbar_arrive(my_x);
      // P as pairs of half floats, and this half's share of the denominator
      uint32_t pw[KT / 2];
      auto exponentials = [&](float m_use) {
        float rs0 = 0.f, rs1 = 0.f;
#pragma unroll
        for (int i = 0; i < KT / 2; ++i) {
          const float p0 = ex2(__uint_as_float(sv[2 * i]) - m_use), p1 = ex2(__uint_as_float(sv[2 * i + 1]) - m_use);
          if (i < 8) rs0 += p0 + p1;
          else rs1 += p0 + p1;
          pw[i] = q8::pack_half(p0, p1);
        }
        return fmaf(rs0, sc0.z, rs1 * sc1.z);
      };
      // taken against the present reference while the other thread's maximum is on its way, and again for rows whose reference moves
      const bool ahead = __all_sync(0xffffffffu, m_ref != -INFINITY);
      float rs = 0.f;
      if (ahead) rs = exponentials(m_ref);
      ok = mbar_wait_spin(my_x, (uint32_t)(t & 1), a.status, 32, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      mx = fmaxf(mx, *max_other);
      mbar_arrive(my_r);
      const bool move = mx > m_ref + RESCALE_STEP || (m_ref == -INFINITY && mx > -INFINITY);
      float corr = 1.f;
      if (move) {
        corr = ex2(m_ref - mx);                                    // 0 when there was no reference yet
        m_ref = mx;
      }
      if (!ahead || move) rs = exponentials((m_ref == -INFINITY) ? 0.f : m_ref);
      l_run = l_run * corr + rs;
      if (t > 0 && __any_sync(0xffffffffu, move)) {
        ok = mbar_wait_spin(&bar_pv[rt], (uint32_t)((t - 1) & 1), a.status, 30, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = hh * HC; c < hh * HC + HC; c += 32) {
          uint32_t ov[32];
          tmem_ld32(lane_addr + O_COL + c, ov);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * corr);
          tmem_st32(lane_addr + O_COL + c, ov);
        }
      }
      // over the first half of S(t): the second thread's words lie over scores of the FIRST thread of the row, which has them in
      // registers since before it left its maximum
      tmem_st16(s_addr + hh * 16, pw);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bar_p[2 * rt + (t & 1)]);
    }
    if (ok && n_tiles > 0) {
      ok = mbar_wait(&bar_o[rt], 0, a.status, 25, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
    }
    // the row's denominator is the two halves' (same reference): through the maxima's places, once the last ones have been read
    if (ok && n_tiles > 0) {
      ok = mbar_wait_spin(my_r, (uint32_t)((n_tiles - 1) & 1), a.status, 33, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        *max_mine = l_run;
        mbar_arrive(my_x);
        ok = mbar_wait_spin(my_x, (uint32_t)(n_tiles & 1), a.status, 34, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) l_run += *max_other;
      }
    }
    if (ok) {
      tc_fence_after();
      bf16* dst = a.out + (size_t)(qs + tok) * a.o_ts + (size_t)(kvh * G + g) * HD;
      const float inv = l_run > 0.f ? 1.f / l_run : l_run;         // nothing seen: 0; NaN stays
#pragma unroll 1
      for (int c = hh * HC; c < hh * HC + HC; c += 32) {
        uint32_t ov[32];
        if (n_tiles > 0) {
          tmem_ld32(lane_addr + O_COL + c, ov);                    // the whole warp loads; rows without a query store nothing
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = 0u;
        }
        if (row_ok) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 pk = __floats2bfloat162_rn(__uint_as_float(ov[i + 2 * e]) * inv, __uint_as_float(ov[i + 2 * e + 1]) * inv);
              w[e] = *reinterpret_cast<const uint32_t*>(&pk);
            }
            *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == SH::MMA_WARP)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(SH::TMEM_COLS) : "memory");
}

int g_row_tiles = 0;

template <int HD, int NR>
cudaError_t launch(const PreArgs& a, int B, int max_q_len, cudaStream_t s) {
  using SH = Shape<HD, NR>;
  static const cudaError_t configured =
      cudaFuncSetAttribute(attention_q8_prefill_kernel<HD, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SH::SMEM);
  if (configured != cudaSuccess) return configured;
  const dim3 grid(ceil_div(max_q_len * (a.H / a.KVH), NR * TQ), a.KVH, B);
  return ts_launch(attention_q8_prefill_kernel<HD, NR>, grid, dim3(SH::THREADS), SH::SMEM, s, a);
}

}  // namespace

TS_API void ts_set_q8_prefill(int row_tiles) { g_row_tiles = row_tiles == 1 || row_tiles == 2 ? row_tiles : 0; }   // for measurements

// Requests of any number of tokens (rows q_start[b] ..).  q, out: rows [H, D] q_ts / o_ts elements apart.
TS_API int ts_attention_q8_prefill(void* out, long long o_ts, const void* q, long long q_ts, const void* k_cache, const void* v_cache,
                                   const float* k_scale, const float* v_scale, const int* block_tables, const int* q_start,
                                   const int* seq_lens, int B, int table_width, int max_q_len, int H, int KVH, int D, int page,
                                   float scale, int window, void* stream) {
  if (B <= 0 || max_q_len <= 0) return 0;
  if (KVH <= 0 || H % KVH != 0 || (D != 64 && D != 128) || page < 16 || page % 16 != 0)
    TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_prefill: H=%d KVH=%d D=%d page=%d is not taken by this kernel", H, KVH, D, page);
  if (B > 65535 || KVH > 65535 || (long long)max_q_len * (H / KVH) > 0x7fffff00LL)
    TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_prefill: %d requests of up to %d tokens, %d kv heads", B, max_q_len, KVH);
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) != 0 || (q_ts & 7) != 0 || (o_ts & 7) != 0)
    TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_prefill: pages and rows of queries and outputs on 16 bytes");
  int* status = ts_attn_status_word();
  if (status == nullptr) TS_REFUSE(TS_ERR_LIMIT, "ts_attention_q8_prefill: no status word");
  const PreArgs a = {(bf16*)out, o_ts, (const bf16*)q, q_ts, {(const unsigned char*)k_cache, (const unsigned char*)v_cache},
                     {k_scale, v_scale}, block_tables, q_start, seq_lens, table_width, H, KVH, page, scale, window, status};
  cudaStream_t s = (cudaStream_t)stream;
  const long long pairs = (long long)ceil_div(max_q_len * (H / KVH), 2 * TQ) * KVH * B;
  const bool two = g_row_tiles ? g_row_tiles == 2 : pairs > ts_sm_count();
  const cudaError_t e = D == 64 ? (two ? launch<64, 2>(a, B, max_q_len, s) : launch<64, 1>(a, B, max_q_len, s))
                                : (two ? launch<128, 2>(a, B, max_q_len, s) : launch<128, 1>(a, B, max_q_len, s));
  if (e != cudaSuccess) TS_REFUSE((int)e, "ts_attention_q8_prefill: %s", cudaGetErrorString(e));
  TS_LAUNCH_CHECK();
}
