// Attention of prompt portions over an 8-bit paged cache (q8_cache.cuh) on the 5th-generation tensor cores: bfloat16 queries, heads
// of 64 or 128, pages of a multiple of 16 tokens, any group size.
//
// Mathematics as in attention_q8_decode.cu: weights P = 2^(t - M), t = score + log2 of the value's scale, on values as they lie in
// the pages; the denominator sums P / scale.  Both products take half floats: keys and values as they are (e4m3 fits whole), queries
// scaled by a power of two a row, P below 2^8.  The scales are constants of 16 keys, so a score costs one fused multiply-add as it would
// without them, and a sum one more for 16 weights.
//
// One block = NR tiles of 128 query rows (a row is a (token, head-in-group) pair of one kv head) over the same keys, 128 a turn.
// Softmax: four warps a row tile, a thread a row = tensor-memory lane, which holds a turn's 128 scores in registers: their maximum (the
// scale of 16 keys is one factor, so that is the maximum of the products, three an instruction, and one multiply-add), then the weights, which
// go back over the scores as pairs of half floats.  One warp issues the products (one lane): S(t) = Q K(t)^T, O += P(t) V(t) with
// P read from tensor memory.  Seven
// warps (eleven where NR = 1) turn the pages' bytes into half floats, 16 rows of keys or values a job: 16 bytes a piece, brought by
// cp.async to a place that its lane alone reads while other rows are converted, stored with the 128-byte swizzle that the products read (values with keys along
// the rows: MN-major).  Rows outside the visible range are zeros.
// NR = 2: a score buffer each, so that the softmax of one row tile runs beside the products of the other; a converted tile serves 256 rows;
// tensor memory is full and a block fills an SM.  NR = 1, for launches of few row tiles, which are as slow as their longest block: two score
// buffers, products two turns ahead; where there are fewer row tiles than half the SMs, a cluster of 2 to 8 blocks cuts the keys of one among
// itself, and every block finishes some of the rows out of its peers' shared memory.
// The reference M moves only when a row's maximum has grown by more than 2^8 since: then O is rescaled in tensor memory.  Every wait is
// bounded; a block that gives up records where, stops, and frees its tensor memory.
//
// NaN: a page whose scale is NaN (either) gives NaN scores, which the rows that do not see it drop by selection; its values are
// finite bytes (writes store zeros under such a scale), so zero weights stay zeros.
#include "mma_utils.cuh"
#include "q8_cache.cuh"
#include "tc_utils.cuh"

namespace {

using namespace tc;

constexpr int TQ = 128, TK = 128, STAGES = 2, SCALE_STAGES = 4, MAX_SPLITS = 8;
constexpr float RESCALE_STEP = 8.f;
constexpr float LOG2E_P = 1.4426950408889634f;

template <int HD, int NR>
struct Shape {
  static constexpr int NB = NR == 1 ? 2 : 1;                       // score buffers of a row tile
  // 16 warps in four warpgroups: softmax (one or two), then the converters and, the last warp, the one that issues the products.  128 registers a
  // thread are there; what the others give back the softmax takes: 256 x 200 + 256 x 56, 128 x 232 + 384 x 88.
  static constexpr int THREADS = 512, SOFT_WARPS = 4 * NR, MMA_WARP = 15, CONV_WARPS = MMA_WARP - SOFT_WARPS;
  static constexpr int SOFT_REGS = NR == 1 ? 232 : 200, OTHER_REGS = NR == 1 ? 88 : 56;
  static constexpr uint32_t Q_BYTES = TQ * HD * 2, KV_BYTES = TK * HD * 2, HALF_Q = TQ * 128, HALF_K = TK * 128;
  static constexpr uint32_t O_COL = NB * TK, ROW_COLS = O_COL + HD; // tensor-memory columns of a row tile: scores, O
  static constexpr uint32_t TMEM_COLS = ROW_COLS * NR <= 256 ? 256 : 512;
  static constexpr int BARS = 4 * STAGES + NR * (2 * NB + 2) + 1;
  // 16 rows of keys or of values are a converter's job; so many jobs of its are on their way from the pages
  static constexpr int AHEAD = 2;
  static constexpr uint32_t JOB_BYTES = 16 * HD;
  static constexpr int O_ROW = HD + 4;                             // floats of a row's sums in shared memory, over the tiles
  static_assert(NR == 2 || (TQ * O_ROW + 2 * TQ) * 4 <= NR * Q_BYTES + 2 * STAGES * KV_BYTES, "sums and references over the tiles");
  static constexpr size_t TILES = NR * Q_BYTES + 2 * STAGES * KV_BYTES + CONV_WARPS * AHEAD * JOB_BYTES;
  // behind the tiles: scales [4][8] float4, scales on their way [converters][AHEAD][2], barriers, the tensor memory's address, the abort flag
  static constexpr size_t SMEM = TILES + SCALE_STAGES * (TK / 16) * 16 + CONV_WARPS * AHEAD * 8 + BARS * 8 + 16;
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
  int window, nsplit;
  int* status;
};

// Instruction descriptor: half x half -> float, M = 128, N = n; A K-major, B K-major or (b_mn) MN-major.
__host__ __device__ constexpr uint32_t instr_half(int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// One lane of the warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// Shared-memory descriptors of tiles with the 128-byte swizzle: the address (and, MN-major, the distance of 64 elements along that dimension)
// in the lower half (K-major: 1, unused); 8-row groups 1,024 bytes apart, the version and the swizzle in the upper one.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr) { return (addr & 0x3FFFF) >> 4; }
template <int ACC>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %5, 0;\n mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}\n"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(DESC_HI), "r"(idesc), "n"(ACC) : "memory");
}
template <int ACC>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %5, 0;\n mov.b64 b, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n"
      ::"r"(d), "r"(a), "r"(b_lo), "r"(DESC_HI), "r"(idesc), "n"(ACC) : "memory");
}

// Registers a thread of the warpgroup gives back, or takes out of what others gave back.
template <int N> __device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
// The largest of three.
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// Block `share` of a cluster of NS finishes rows share * TQ / NS .. of their row tile: 128 threads, four columns each, the sums of every
// block out of its shared memory, in the order of the shares.  (Eight loads of a thread on their way at a time: one piece at a time
// cost 5 us more.)
template <int HD, int NS>
__device__ __forceinline__ void merge_shares(const PreArgs& a, const unsigned char* smem, int tid, int share, int rows, int qs, int row0, int kvh,
                                             int G) {
  constexpr int O_ROW = Shape<HD, 1>::O_ROW, PB = MAX_SPLITS / NS, CPR = HD / 4, FIRST_ROWS = TQ / CPR;
  const float* o_s = reinterpret_cast<const float*>(smem);
  const float* m_s = o_s + TQ * O_ROW;
  const int d = tid % CPR * 4;
  for (int r0 = share * (TQ / NS) + tid / CPR; r0 < (share + 1) * (TQ / NS) && r0 < rows; r0 += FIRST_ROWS * PB) {
    float m1[PB][NS], l1[PB][NS];
    float4 x[PB][NS];
#pragma unroll
    for (int p = 0; p < PB; ++p)
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int r = r0 + p * FIRST_ROWS;
        m1[p][i] = ld_peer_f32(peer_shared(m_s + r, i));
        l1[p][i] = ld_peer_f32(peer_shared(m_s + TQ + r, i));
        x[p][i] = ld_peer_v4(peer_shared(o_s + r * O_ROW + d, i));
      }
#pragma unroll
    for (int p = 0; p < PB; ++p) {
      const int r = r0 + p * FIRST_ROWS, row = row0 + r;
      float M = -INFINITY, L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NS; ++i) M = fmaxf(M, m1[p][i]);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        // (no reference: the share saw nothing, and weighs nothing, or NaN alone)
        const float f = m1[p][i] == -INFINITY ? l1[p][i] : ex2(m1[p][i] - M);
        L = fmaf(l1[p][i], f, L);
        acc.x = fmaf(x[p][i].x, f, acc.x);
        acc.y = fmaf(x[p][i].y, f, acc.y);
        acc.z = fmaf(x[p][i].z, f, acc.z);
        acc.w = fmaf(x[p][i].w, f, acc.w);
      }
      const float inv = L > 0.f ? 1.f / L : L;                     // nothing seen: 0; NaN stays
      bf16* dst = a.out + (size_t)(qs + row / G) * a.o_ts + (size_t)(kvh * G + row % G) * HD + d;
      if (r < rows) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
    }
  }
}

template <int HD, int NR>
__global__ void __launch_bounds__(Shape<HD, NR>::THREADS, 1) attention_q8_prefill_kernel(const PreArgs a) {
  using SH = Shape<HD, NR>;
  constexpr uint32_t KV_BYTES = SH::KV_BYTES, HALF_K = SH::HALF_K, HALF_Q = SH::HALF_Q, ROW_COLS = SH::ROW_COLS, O_COL = SH::O_COL;
  constexpr int ROWS = NR * TQ, NB = SH::NB, GROUPS = TK / 16;
  pdl_launch_dependents();
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* q_s = smem;                                       // [NR][HD / 64][128][128 B]
  unsigned char* k_s = q_s + NR * SH::Q_BYTES;                     // [STAGES][HD / 64][128][128 B]
  unsigned char* v_s = k_s + STAGES * KV_BYTES;
  unsigned char* raw_s = v_s + STAGES * KV_BYTES;                  // [converters][AHEAD][pieces a lane][32 lanes][16 B]
  float4* scale_s = reinterpret_cast<float4*>(raw_s + SH::CONV_WARPS * SH::AHEAD * SH::JOB_BYTES);        // [SCALE_STAGES][GROUPS]
  float* raw_scale = reinterpret_cast<float*>(scale_s + SCALE_STAGES * GROUPS);                           // [converters][AHEAD][2]
  uint64_t* full_k = reinterpret_cast<uint64_t*>(raw_scale + SH::CONV_WARPS * SH::AHEAD * 2);
  uint64_t* empty_k = full_k + STAGES;
  uint64_t* full_v = empty_k + STAGES;
  uint64_t* empty_v = full_v + STAGES;
  uint64_t* bar_s = empty_v + STAGES;                              // [NR][NB]: that score buffer is complete
  uint64_t* bar_p = bar_s + NB * NR;                               // [NR][NB]: all rows have read S(t) and written P(t)
  uint64_t* bar_pv = bar_p + NB * NR;                              // [NR]: an O product is complete
  uint64_t* bar_o = bar_pv + NR;                                   // [NR]: the last one
  uint64_t* bar_q = bar_o + NR;                                    // the queries are in place
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_q + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int nsplit = NR == 1 ? a.nsplit : 1, share = blockIdx.x % nsplit, block_row = blockIdx.x / nsplit;
  const int b = blockIdx.z, kvh = blockIdx.y, G = a.H / a.KVH;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((smem_u32(smem) & 1023u) != 0) {                             // the swizzled tiles need 1024-byte alignment
    if (tid == 0) atomicCAS(a.status, 0, 29);
    return;
  }
  pdl_wait();                                                      // what it reads is written by kernels before
  const int qs = a.q_start[b], q_len = a.q_start[b + 1] - qs, seq_len = a.seq_lens[b];
  const int n_rows = q_len * G, n_blocks = (n_rows + ROWS - 1) / ROWS;
  if (block_row >= n_blocks) return;                               // (the whole cluster)
  const int row0 = (n_blocks - 1 - block_row) * ROWS;              // longest blocks first
  const int prefix = seq_len - q_len;
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_k[s], GROUPS);
      mbar_init(&empty_k[s], 1);
      mbar_init(&full_v[s], GROUPS);
      mbar_init(&empty_v[s], 1);
    }
    for (int r = 0; r < NR; ++r) {
      for (int i = 0; i < NB; ++i) {
        mbar_init(&bar_s[NB * r + i], 2);                          // the product's end, and the issuing thread, which saw the scales
        mbar_init(&bar_p[NB * r + i], TQ);
      }
      mbar_init(&bar_pv[r], 1);
      mbar_init(&bar_o[r], 1);
    }
    mbar_init(bar_q, SH::SOFT_WARPS * 32);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == SH::MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(SH::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int last_row = min(row0 + ROWS, n_rows) - 1;
  const int key_hi = prefix + last_row / G;                        // the last key that any row sees, and the first
  const int key_lo = a.window > 0 ? max(0, prefix + row0 / G - a.window + 1) : 0;
  const int all_tiles = (seq_len > 0 && key_hi >= key_lo) ? (key_hi - (key_lo & ~15)) / TK + 1 : 0;
  // this block's turns of them
  const int first_tile = (int)((long long)all_tiles * share / nsplit);
  const int n_tiles = (int)((long long)all_tiles * (share + 1) / nsplit) - first_tile;
  const int j_lo = (key_lo & ~15) + first_tile * TK, j_hi = min(key_hi, j_lo + n_tiles * TK - 1);

  const int rt = warp >> 2, lane_row = tid & (TQ - 1);             // a softmax thread's row tile and row
  const bool softmax = warp < SH::SOFT_WARPS;
  const int row = row0 + tid;
  const bool row_ok = softmax && row < n_rows;
  const int tok = row_ok ? row / G : 0, g = row_ok ? row % G : 0;
  const int pos = row_ok ? prefix + tok : -1;

  // (a warpgroup takes or gives as one: its four warps at the same instruction)
  if (softmax) take_registers<SH::SOFT_REGS>();
  else give_registers<SH::OTHER_REGS>();

  if (softmax) {
    // ================= softmax: a thread a row = tensor-memory lane =================
    // Q rows -> shared memory as half floats, K-major with the 128-byte swizzle (16-byte piece c of row r at c ^ (r & 7))
    float factor = 0.f;
    {
      const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)(qs + tok) * a.q_ts + (size_t)(kvh * G + g) * HD);
      uint4 v[HD / 8];
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) v[c] = row_ok ? src[c] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) {
        const unsigned w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          amax = fmaxf(amax, fmaxf(q8::abs_or_inf(__uint_as_float(w[i] << 16)), q8::abs_or_inf(__uint_as_float(w[i] & 0xffff0000u))));
      }
      // (the factor is positive: a negative scale turns the queries)
      float to_half = q8::query_to_half(amax, fabsf(a.scale) * LOG2E_P, factor);
      if (a.scale < 0.f) to_half = -to_half;
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) {
        const unsigned w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
        unsigned h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          h[i] = q8::pack_half(__uint_as_float(w[i] << 16) * to_half, __uint_as_float(w[i] & 0xffff0000u) * to_half);
        *reinterpret_cast<uint4*>(q_s + rt * SH::Q_BYTES + (c >> 3) * HALF_Q + lane_row * 128 + (((c & 7) ^ (lane_row & 7)) << 4)) =
            make_uint4(h[0], h[1], h[2], h[3]);
      }
      fence_async_smem();
      mbar_arrive(bar_q);
    }
    float m_ref = -INFINITY, l_run = 0.f;
    const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16) + rt * ROW_COLS;
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      const uint32_t s_addr = lane_addr + (t % NB) * TK;
      ok = mbar_wait_spin(&bar_s[NB * rt + t % NB], (uint32_t)((t / NB) & 1), a.status, 22, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const int j0 = j_lo + t * TK;
      const float4* sc = scale_s + (t % SCALE_STAGES) * GROUPS;
      // keys wholly before every row of the warp (the common case away from the diagonal) need no mask
      const bool all_visible = __all_sync(0xffffffffu, (j0 + TK - 1 <= pos) && (a.window <= 0 || j0 > pos - a.window));
      const int see_lo = a.window > 0 ? max(0, pos - a.window + 1 - j0) : 0;       // the row sees keys see_lo .. see_lo + see_n of the turn
      const unsigned see_n = (unsigned)max(0, min(TK, pos + 1 - j0) - see_lo);
      bool move = false;
      float corr = 1.f, rs = 0.f;
      auto new_reference = [&](float mx) {
        move = mx > m_ref + RESCALE_STEP || (m_ref == -INFINITY && mx > -INFINITY);
        if (move) {
          corr = ex2(m_ref - mx);                                  // 0 when there was no reference yet
          m_ref = mx;
        }
        return m_ref == -INFINITY ? 0.f : m_ref;
      };
      // a turn whose keys every row of the warp sees
      auto whole_turn = [&]() {
        uint32_t sv[TK];
#pragma unroll
        for (int c = 0; c < TK / 32; ++c) tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(sv + c * 32));
        tmem_wait_ld();
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < GROUPS; ++h) {
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 16; i += 2)
            top[i >> 1 & 1] = max3(top[i >> 1 & 1], __uint_as_float(sv[h * 16 + i]), __uint_as_float(sv[h * 16 + i + 1]));
          const float4 x = sc[h];
          mx = fmaxf(mx, fmaf(fmaxf(top[0], top[1]), x.x * factor, x.y));
        }
        const float m_use = new_reference(mx);
#pragma unroll
        for (int h = 0; h < GROUPS; ++h) {
          const float4 x = sc[h];
          const float f = x.x * factor, add = x.y - m_use;
          float part[2] = {0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float p0 = ex2(fmaf(__uint_as_float(sv[h * 16 + i]), f, add));
            const float p1 = ex2(fmaf(__uint_as_float(sv[h * 16 + i + 1]), f, add));
            part[0] += p0;
            part[1] += p1;
            sv[h * 8 + i / 2] = q8::pack_half(p0, p1);             // (its place has been read)
          }
          rs = fmaf(part[0] + part[1], x.z, rs);
          if (h % 4 == 3) tmem_st32(s_addr + (h / 4) * 32, *reinterpret_cast<const uint32_t(*)[32]>(sv + (h / 4) * 32));
        }
      };
      // a turn at an edge of what is seen: 32 scores a turn of two loops, which stay loops (few turns are such, and code that is run once is
      // mostly waited for)
      auto edge_turn = [&]() {
        auto seen = [&](int c) {                                   // of keys 32 c ..: a bit each
          const int lo = min(max(see_lo - 32 * c, 0), 32), hi = min(max(see_lo + (int)see_n - 32 * c, 0), 32);
          return (uint32_t)((1ull << hi) - 1) & ~(uint32_t)((1ull << lo) - 1);
        };
        float mx = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < TK / 32; ++c) {
          uint32_t sv[32];
          tmem_ld32(s_addr + c * 32, sv);
          const uint32_t bits = seen(c);
          tmem_wait_ld();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i += 2)
              top = max3(top, bits >> (h * 16 + i) & 1 ? __uint_as_float(sv[h * 16 + i]) : -INFINITY,
                         bits >> (h * 16 + i + 1) & 1 ? __uint_as_float(sv[h * 16 + i + 1]) : -INFINITY);
            const float4 x = sc[2 * c + h];
            if (top > -INFINITY) mx = fmaxf(mx, fmaf(top, x.x * factor, x.y));            // (nothing seen: no maximum, whatever the factor)
          }
        }
        const float m_use = new_reference(mx);
#pragma unroll 1
        for (int c = 0; c < TK / 32; ++c) {
          uint32_t sv[32], pw[16];
          tmem_ld32(s_addr + c * 32, sv);
          const uint32_t bits = seen(c);
          tmem_wait_ld();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 x = sc[2 * c + h];
            const float f = x.x * factor, add = x.y - m_use;
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float p0 = bits >> (h * 16 + i) & 1 ? ex2(fmaf(__uint_as_float(sv[h * 16 + i]), f, add)) : 0.f;
              const float p1 = bits >> (h * 16 + i + 1) & 1 ? ex2(fmaf(__uint_as_float(sv[h * 16 + i + 1]), f, add)) : 0.f;
              part += p0 + p1;
              pw[h * 8 + i / 2] = q8::pack_half(p0, p1);
            }
            rs = fmaf(part, x.z, rs);
          }
          tmem_st16(s_addr + c * 16, pw);                          // over scores that have been read
        }
      };
      if (all_visible) whole_turn();
      else edge_turn();
      l_run = l_run * corr + rs;
      if (t > 0 && __any_sync(0xffffffffu, move)) {
        if (NB == 2) {                                             // (one buffer: S(t) was issued behind the product before, and is complete)
          ok = mbar_wait_spin(&bar_pv[rt], (uint32_t)((t - 1) & 1), a.status, 30, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
        }
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t ov[32];
          tmem_ld32(lane_addr + O_COL + c, ov);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * corr);
          tmem_st32(lane_addr + O_COL + c, ov);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bar_p[NB * rt + t % NB]);
    }
    if (ok && n_tiles > 0) {
      ok = mbar_wait(&bar_o[rt], 0, a.status, 25, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok && nsplit > 1) {
      // The row's sums, for whichever block of the cluster finishes it: over the tiles, which nobody reads any more, and which all rows have
      // written: the last product has seen every query, and in a share without turns, where there is no product, the rows meet here.
      // (A query stored late would lie in another row's sums, and a NaN in it counts even at no weight.)
      if (n_tiles == 0) asm volatile("bar.sync 1, %0;" ::"n"(TQ) : "memory");
      tc_fence_after();
      float* dst = reinterpret_cast<float*>(smem) + lane_row * SH::O_ROW;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t ov[32];
        if (n_tiles > 0) {
          tmem_ld32(lane_addr + O_COL + c, ov);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
      }
      dst = reinterpret_cast<float*>(smem) + TQ * SH::O_ROW + lane_row;
      dst[0] = m_ref;
      dst[TQ] = l_run;
    } else if (ok) {
      tc_fence_after();
      bf16* dst = a.out + (size_t)(qs + tok) * a.o_ts + (size_t)(kvh * G + g) * HD;
      const float inv = l_run > 0.f ? 1.f / l_run : l_run;         // nothing seen: 0; NaN stays
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
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
  } else if (warp != SH::MMA_WARP) {
    // ================= converters: each warp takes every CONV_WARPS-th job, 16 rows of keys (and their scales) or of values =================
    constexpr int CPR = HD / 16, NP = CPR / 2, RPP = 32 / CPR;     // 16-byte pieces of a row; pieces a lane takes; rows the lanes cover with one each
    // A lane's piece c16 of rows r0, r0 + RPP, ...: eight neighbouring lanes have four pieces of two rows, whose stores (every other piece of a
    // line of the converted tile, swapped by the row's number) then go to eight different places of a line.
    const int cw = warp - SH::SOFT_WARPS;
    const int c16 = HD == 128 ? (lane & 3) + (lane >> 1 & 4) : lane & 3, r0 = HD == 128 ? (lane >> 2 & 1) + (lane >> 4) * 2 : lane >> 2;
    const int* table = a.block_tables + (size_t)b * a.table_width;
    const int n_jobs = n_tiles * 2 * GROUPS;
    // the page and the place in it of 16 keys, a lane, of 512 rows: -1 outside; fetched that many rows ahead
    int pg = -1, in_page = 0, pg_next, in_next, block = -1;
    auto fetch_pages = [&](int blk) {
      const int j = j_lo + blk * 512 + lane * 16, lp = j / a.page;
      in_next = j - lp * a.page;
      pg_next = (j <= j_hi && lp < a.table_width) ? table[lp] : -1;
    };
    fetch_pages(0);
    // a job's rows from its page, asynchronously: a lane's pieces go to a place of its own, which it alone reads
    unsigned char* raw = raw_s + cw * SH::AHEAD * SH::JOB_BYTES + lane * 16;
    float* raw_sc = raw_scale + cw * SH::AHEAD * 2;
    auto issue = [&](int job, int slot) {
      if (job < n_jobs) {
        const int t = job / (2 * GROUPS), kv = job / GROUPS & 1, grp = job % GROUPS;
        if (t / 4 != block) {
          block = t / 4;
          pg = pg_next;
          in_page = in_next;
          fetch_pages(block + 1);
        }
        const int p = __shfl_sync(0xffffffffu, pg, (t & 3) * GROUPS + grp), in = __shfl_sync(0xffffffffu, in_page, (t & 3) * GROUPS + grp);
        const size_t at = (size_t)max(p, 0) * a.KVH + kvh;
        const unsigned char* src = (kv ? a.cache[1] : a.cache[0]) + (at * a.page + in + r0) * HD + c16 * 16;
        const int j0 = j_lo + t * TK + grp * 16 + r0;
#pragma unroll
        for (int i = 0; i < NP; ++i)
          cp_async_16(raw + slot * SH::JOB_BYTES + i * 512, src + i * RPP * HD, p >= 0 && j0 + i * RPP >= key_lo && j0 + i * RPP <= j_hi);
        if (kv == 0 && lane < 2) cp_async_4(raw_sc + slot * 2 + lane, (lane == 0 ? a.scales[0] : a.scales[1]) + at, p >= 0);
      }
      cp_async_commit();
    };
#pragma unroll 1
    for (int i = 0; i < SH::AHEAD; ++i) issue(cw + i * SH::CONV_WARPS, i);
    bool ok = true;
    for (int job = cw, slot = 0; job < n_jobs; job += SH::CONV_WARPS, slot = (slot + 1) % SH::AHEAD) {
      const int t = job / (2 * GROUPS), kv = job / GROUPS & 1, grp = job % GROUPS, st = t % STAGES;
      if (t >= STAGES) {
        ok = mbar_wait(kv ? &empty_v[st] : &empty_k[st], (uint32_t)((t / STAGES - 1) & 1), a.status, kv ? 27 : 24, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      cp_async_wait<SH::AHEAD - 1>();
      // columns 16 c16 .. of the row: half c16 / 4 of the head, pieces 2 (c16 & 3) and the next
      unsigned char* line = (kv ? v_s : k_s) + st * KV_BYTES + (c16 >> 2) * HALF_K + (grp * 16 + r0) * 128;
      const int lo_at = (2 * (c16 & 3) ^ (r0 & 7)) << 4;           // (the next piece's is this one's last bit turned; four rows on, the third)
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const uint4 piece = *reinterpret_cast<const uint4*>(raw + slot * SH::JOB_BYTES + i * 512);
        uint4 lo, hi;
        q8::halves_of(piece.x, lo.x, lo.y);
        q8::halves_of(piece.y, lo.z, lo.w);
        q8::halves_of(piece.z, hi.x, hi.y);
        q8::halves_of(piece.w, hi.z, hi.w);
        const int swap = lo_at ^ (i * RPP % 8 << 4);
        *reinterpret_cast<uint4*>(line + i * RPP * 128 + swap) = lo;
        *reinterpret_cast<uint4*>(line + i * RPP * 128 + (swap ^ 16)) = hi;
      }
      if (kv == 0) {
        __syncwarp();                                              // (lane 1 brought the values' scale)
        if (lane == 0) {
          const float ks = raw_sc[slot * 2], vs = raw_sc[slot * 2 + 1];
          // (score factor, log2 of the value's scale, its inverse) of the 16 keys
          scale_s[(t % SCALE_STAGES) * GROUPS + grp] =
              make_float4(vs != vs ? vs : ks, (float)((int)(__float_as_uint(vs) >> 23) - 127), q8::inverse_scale(vs), 0.f);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(kv ? &full_v[st] : &full_k[st]);
      issue(job + SH::AHEAD * SH::CONV_WARPS, slot);
    }
    cp_async_wait<0>();
  } else {
    // ================= product issue, one lane =================
    if (n_tiles > 0) {
      // The whole warp walks the loop and waits; one elected lane issues.  (Descriptors stay uniform values that way: their upper halves are
      // constants, the lower ones advance by constants.)
      const bool one = elect_one();
      const uint32_t q_lo = desc_lo(smem_u32(q_s)) | 1u << 16, k_lo = desc_lo(smem_u32(k_s)) | 1u << 16, v_lo = desc_lo(smem_u32(v_s)) | ((HALF_K >> 4) << 16);
      auto issue_s = [&](int r, int t) {
        constexpr uint32_t idesc = instr_half(TK, false);
        const uint32_t qa = q_lo + r * (SH::Q_BYTES >> 4), ka = k_lo + (t % STAGES) * (KV_BYTES >> 4), d = tmem + r * ROW_COLS + (t % NB) * TK;
        if (one) {
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t aq = qa + ((ks >> 2) * HALF_Q + (ks & 3) * 32 >> 4), ak = ka + ((ks >> 2) * HALF_K + (ks & 3) * 32 >> 4);
            if (ks == 0) mma_ss<0>(d, aq, ak, idesc);
            else mma_ss<1>(d, aq, ak, idesc);
          }
          umma_commit(&bar_s[NB * r + t % NB]);
          mbar_arrive(&bar_s[NB * r + t % NB]);
          if (r == NR - 1) umma_commit(&empty_k[t % STAGES]);
        }
      };
      auto issue_o = [&](int r, int t) {
        constexpr uint32_t idesc = instr_half(HD, true);
        const uint32_t va = v_lo + (t % STAGES) * (KV_BYTES >> 4), d = tmem + r * ROW_COLS + O_COL, pa = tmem + r * ROW_COLS + (t % NB) * TK;
        if (one) {
          if (t == 0) mma_ts<0>(d, pa, va, idesc);
          else mma_ts<1>(d, pa, va, idesc);
#pragma unroll
          for (int kk = 1; kk < TK / 16; ++kk) mma_ts<1>(d, pa + kk * 8, va + (kk * 16 * 128 >> 4), idesc);
          if (r == NR - 1) umma_commit(&empty_v[t % STAGES]);
          umma_commit(&bar_pv[r]);
          if (t + 1 == n_tiles) umma_commit(&bar_o[r]);
        }
      };
      bool ok = mbar_wait(bar_q, 0, a.status, 20, abort_flag);
      for (int t = 0; t < NB && t < n_tiles && ok; ++t) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full_k[t % STAGES], 0, a.status, 21, abort_flag));
        if (!ok) break;
        tc_fence_after();
        for (int r = 0; r < NR; ++r) issue_s(r, t);
      }
      for (int t = 0; t < n_tiles && ok; ++t)
        for (int r = 0; r < NR && ok; ++r) {
          ok = mbar_wait_spin(&bar_p[NB * r + t % NB], (uint32_t)((t / NB) & 1), a.status, 26, abort_flag);
          if (ok && r == 0) ok = mbar_wait(&full_v[t % STAGES], (uint32_t)((t / STAGES) & 1), a.status, 23, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          issue_o(r, t);
          if (t + NB < n_tiles) {
            if (r == 0) ok = __all_sync(0xffffffffu, mbar_wait(&full_k[(t + NB) % STAGES], (uint32_t)(((t + NB) / STAGES) & 1), a.status, 28, abort_flag));
            if (!ok) break;
            tc_fence_after();
            issue_s(r, t + NB);                                    // over P(t), behind the product that reads it
          }
        }
    }
  }
  if (NR == 1 && nsplit > 1) {
    // Block `share` finishes its share of the rows out of its peers' shared memory, in the order of the shares.
    cluster_sync_all();
    if (softmax) {
      const int rows_here = n_rows - row0;
      if (nsplit == 2) merge_shares<HD, 2>(a, smem, tid, share, rows_here, qs, row0, kvh, G);
      else if (nsplit == 4) merge_shares<HD, 4>(a, smem, tid, share, rows_here, qs, row0, kvh, G);
      else merge_shares<HD, 8>(a, smem, tid, share, rows_here, qs, row0, kvh, G);
    }
    cluster_sync_all();                                            // no block leaves while a peer still reads it
  }
  tc_fence_before();
  __syncthreads();
  if (warp == SH::MMA_WARP)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(SH::TMEM_COLS) : "memory");
}

int g_row_tiles = 0, g_splits = 0;

// Whether the device holds a block of the instance.
template <int HD, int NR>
bool prepare_kernel() {
  using SH = Shape<HD, NR>;
  constexpr int SOFT = SH::SOFT_WARPS * 32;
  static_assert(SOFT * SH::SOFT_REGS + (SH::THREADS - SOFT) * SH::OTHER_REGS <= SH::THREADS * 128, "more registers than the block has");
  static const bool ready = [] {
    // the split of registers counts on 128 a thread at launch: with fewer a warpgroup would wait for what nobody gives
    cudaFuncAttributes attr;
    const bool ok = cudaFuncGetAttributes(&attr, attention_q8_prefill_kernel<HD, NR>) == cudaSuccess && attr.numRegs == 128 &&
                    cudaFuncSetAttribute(attention_q8_prefill_kernel<HD, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SH::SMEM) == cudaSuccess;
    cudaGetLastError();                                            // a refusal is an answer, not an error
    return ok;
  }();
  return ready;
}

template <int HD, int NR>
cudaError_t launch(const PreArgs& a, int B, int max_q_len, cudaStream_t s) {
  using SH = Shape<HD, NR>;
  const dim3 grid(ceil_div(max_q_len * (a.H / a.KVH), NR * TQ) * a.nsplit, a.KVH, B);
  return ts_launch_cluster(attention_q8_prefill_kernel<HD, NR>, dim3(a.nsplit, 1, 1), grid, dim3(SH::THREADS), SH::SMEM, s, a);
}

// How many clusters of n blocks of one row tile the chip holds at once (0: none).
template <int HD>
int clusters_that_fit(int n) {
  static int known[MAX_SPLITS + 1];
  int& k = known[n];
  if (k == 0) {
    using SH = Shape<HD, 1>;
    k = -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n, 1, 1);
    cfg.blockDim = dim3(SH::THREADS);
    cfg.dynamicSmemBytes = SH::SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)n;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (prepare_kernel<HD, 1>() &&
        cudaOccupancyMaxActiveClusters(&clusters, attention_q8_prefill_kernel<HD, 1>, &cfg) == cudaSuccess && clusters >= 1)
      k = clusters;
    cudaGetLastError();                                            // a refusal is an answer, not an error
  }
  return k < 0 ? 0 : k;
}

// About how many times the longest block's time a launch of n blocks takes, whose lengths fall evenly from 1 to `least`: the work over the
// SMs, or r + 1 of the blocks that are the longest left when an SM takes its (r + 1)th.
double launch_time(long long n, double least) {
  const double sms = ts_sm_count();
  double t = n * (1.0 + least) / 2.0 / sms;
  for (int r = 0; r < n / sms && r < 64; ++r) {
    const double v = (r + 1) * (1.0 - (1.0 - least) * (r * sms / n));
    if (v > t) t = v;
  }
  return t;
}

}  // namespace

// For measurements: row tiles a block (1, 2), and blocks that cut its keys (1, 2, 4, 8, with one row tile); 0: by the rule.
TS_API void ts_set_q8_prefill(int row_tiles) { g_row_tiles = row_tiles == 1 || row_tiles == 2 ? row_tiles : 0; }
TS_API void ts_set_q8_prefill_splits(int splits) { g_splits = splits == 1 || splits == 2 || splits == 4 || splits == 8 ? splits : 0; }

// Requests of any number of tokens (rows q_start[b] ..).  q, out: rows [H, D] q_ts / o_ts elements apart.
TS_API int ts_attention_q8_prefill(const void* record, void* stream) {
  const q8::AttendCall& c = *(const q8::AttendCall*)record;
  const int B = c.B, max_q_len = c.max_q_len, max_seq_len = c.max_seq_len, H = c.H, KVH = c.KVH, D = c.D, page = c.page, window = c.window;
  const long long o_ts = c.o_ts, q_ts = c.q_ts;
  const void *const k_cache = c.k_cache, *const v_cache = c.v_cache, *const q = c.q;
  void* const out = c.out;
  if (B <= 0 || max_q_len <= 0) return 0;
  if (KVH <= 0 || H % KVH != 0 || (D != 64 && D != 128) || page < 16 || page % 16 != 0)
    TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_prefill: H=%d KVH=%d D=%d page=%d is not taken by this kernel", H, KVH, D, page);
  if (B > 65535 || KVH > 65535 || (long long)max_q_len * (H / KVH) > 0x7fffff00LL)
    TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_prefill: %d requests of up to %d tokens, %d kv heads", B, max_q_len, KVH);
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) != 0 || (q_ts & 7) != 0 || (o_ts & 7) != 0)
    TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_prefill: pages and rows of queries and outputs on 16 bytes");
  if (!(D == 64 ? prepare_kernel<64, 1>() && prepare_kernel<64, 2>() : prepare_kernel<128, 1>() && prepare_kernel<128, 2>()))
    TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_prefill: the device does not hold a block");
  int* status = ts_attn_status_word();
  if (status == nullptr) TS_REFUSE(TS_ERR_LIMIT, "ts_attention_q8_prefill: no status word");
  PreArgs a = {(bf16*)out, o_ts, (const bf16*)q, q_ts, {(const unsigned char*)k_cache, (const unsigned char*)v_cache},
               {c.k_scale, c.v_scale}, c.block_tables, c.q_start, c.seq_lens, c.table_width, H, KVH, page, c.scale, window, 1, status};
  cudaStream_t s = (cudaStream_t)stream;
  // Two row tiles a block or one: a turn of 128 keys takes a block of two 1.64 times as long (4,750 against 2,900 cycles), so it is two where half
  // the blocks more than make up for that (us, one / two: 28 heads over 4, 4,096 tokens 194 / 169, 2,048 63 / 71, 1,024 30 / 32, 2,048 behind
  // 4,000 225 / 215; 40 over 8, 512 behind 4,000 109 / 98; 12 over 2, 2,048 31 / 49).
  // A cluster of 2, 4 or 8 blocks of one row tile where all of them run at once and the turns that a block is spared are worth the merge (8,600
  // cycles) and beat both: a block more for an SM costs it 10 us and more, however short (us, one / 2 / 4 / 8: 12 heads over 2, 64 tokens
  // behind 2,000, 6 row tiles, 32 / 24 / 18 / 15; behind 16,000 186 / 102 / 58 / 34; 512 behind 4,000, 48 row tiles, 60 / 39 / 48 / 68; 512 alone
  // 13.4 / 14.1 / 24 / 48; 1,024 alone, 96 row tiles, 19 / 27 / 39 / 84).
  const int rows = max_q_len * (H / KVH);
  const double reach = max_seq_len < 1 ? 1 : max_seq_len, sees = window > 0 && window < reach ? window : reach;
  const double before = max_q_len < reach ? reach - max_q_len : 0, least = (before < sees ? before : sees) / sees;
  const double longest = (sees / TK + 1) * 2900;
  const long long row_tiles = (long long)ceil_div(rows, TQ) * KVH * B;
  const double t_one = launch_time(row_tiles, least), t_two = launch_time((long long)ceil_div(rows, 2 * TQ) * KVH * B, least) * 1.64;
  const bool two = g_row_tiles ? g_row_tiles == 2 : t_two < t_one;
  if (g_splits && !two) a.nsplit = g_splits;
  else if (!g_splits && g_row_tiles != 2 && ts_clusters_enabled()) {
    double best = (two ? t_two : t_one) * longest;
    for (int n = 2; n <= MAX_SPLITS && row_tiles * n <= ts_sm_count(); n *= 2)
      if (longest / n + 8600 < best && row_tiles <= (D == 64 ? clusters_that_fit<64>(n) : clusters_that_fit<128>(n))) {
        best = longest / n + 8600;
        a.nsplit = n;
      }
  }
  const bool pair = two && a.nsplit == 1;
  const cudaError_t e = D == 64 ? (pair ? launch<64, 2>(a, B, max_q_len, s) : launch<64, 1>(a, B, max_q_len, s))
                                : (pair ? launch<128, 2>(a, B, max_q_len, s) : launch<128, 1>(a, B, max_q_len, s));
  if (e != cudaSuccess) TS_REFUSE((int)e, "ts_attention_q8_prefill: %s", cudaGetErrorString(e));
  TS_LAUNCH_CHECK();
}
