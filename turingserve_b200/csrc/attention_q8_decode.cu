// Attention of single tokens over an 8-bit paged cache (q8_cache.cuh): bfloat16 queries, heads of 64 or 128, up to 16
// query heads a kv head, pages of any size.
//
// Mathematics.  Key j of a request has the score s_j = scale * log2(e) * (q . k8_j) * ks_j and the value v8_j * vs_j, the scales
// powers of two.  With t_j = s_j + log2(vs_j) and a reference M >= every t_j,
//   out = sum_j 2^(t_j - M) v8_j / sum_j 2^(t_j - M) / vs_j :
// one exponential a key gives the weight of the value as it lies in the page, and the denominator takes it back to the
// softmax's with an exact factor.  So both products run on what the pages hold, turned to half floats (exact for e4m3, one
// instruction for two values): the queries as half floats too, each head scaled by a power of two to 128..256 (a bfloat16 fits
// whole down to 2^-21 of the head's largest), the weights, at most 1, rounded to 2^-11 (2^-25 of the largest for the
// smallest).  Scales span 2^-50..2^50, so a weight that vanishes here is below 2^-26 of the softmax's denominator.
//
// Layout.  Keys are the 16 rows of mma.sync m16n8k16 and heads its 8 columns (scores as K Q^T, outputs as V^T P^T): a group of up to
// 8 heads leaves no row idle, half the instructions of heads on the rows.  A thread's four bytes of a key row, as ldmatrix
// brings them, are two pairs of columns of the A operand under an order of the head's columns that the queries share; value
// bytes come transposed in pairs, one byte permutation puts two keys of a column side by side.
//
// Work.  One block of four warps a (split, kv head, request); every warp walks tiles of 32 keys of its own with a ring of three
// stages filled by its own cp.async (16 bytes a lane, rows outside the visible range filled with zeros): no barrier and
// no other warp in the loop.  The warps' sums meet in shared memory; the splits' in a cluster's distributed shared memory
// where the blocks of a request and kv head form one, else a second kernel sums what they left in scratch.
//
// What bounds it: long contexts the memory (1 request of 100,001 keys over 8 kv heads of 128 38 us, 5.4 TB/s; 128 of 3,000..4,096 over
// 4 85 us, 5.5 TB/s; 64 of 4,100..8,192 80 us, 5.1 TB/s, the SMs with two of its 256 blocks being the last), short ones the chain launch,
// table, rows, a tile or two, merge (1 request of 57 keys 3.2 us, 8 of 2,048 over 2 kv heads 6.6).  Measured beside it: two stages (twelve
// warps an SM instead of eight) 105 us at one block a pair of the 64 requests and 77 to 80 at three and more, but 28 against 23 for 64 of
// 1,024..2,048; boxes by TMA, whose rows a lane issues for all, 89 against 81.
#include "mma_utils.cuh"
#include "q8_cache.cuh"

namespace {

using namespace q8;

constexpr int WARPS = 4, THREADS = WARPS * 32, TILE = 32, STAGES = 3;
constexpr float LOG2E_Q8 = 1.4426950408889634f;

struct DecArgs {
  bf16* out;
  long long o_ts;
  const bf16* q;
  long long q_ts;
  const unsigned char* cache[2];
  const float* scales[2];
  const int* block_tables;
  const int* q_start;
  const int* seq_lens;
  float* part;                   // [B][KVH][nsplit][G][D] sums, then [B][KVH][nsplit][G][2] (reference, denominator)
  int B, table_width, H, KVH, page;
  float scale;
  int window, nsplit, cluster, early;
};

__device__ __forceinline__ unsigned transpose8x8(unsigned a) {
  unsigned r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A stage: key rows, value rows (32 of D bytes each), their scales.
template <int D>
struct Stage {
  static constexpr int TILE_BYTES = TILE * D;
  static constexpr int BYTES = 2 * TILE_BYTES + 2 * TILE * 4;
  static constexpr int WARP_BYTES = STAGES * BYTES;
  static constexpr size_t SMEM = (size_t)WARPS * WARP_BYTES;
  static constexpr int O_ROW = D + 4;                            // floats of a head's sums in shared memory
};
// Byte offset of 16-byte piece c of a tile's row: pieces of a 128-byte line (one row of 128, two of 64) swapped by the line's number,
// so that eight rows' pieces lie in different banks.
template <int D>
__device__ __forceinline__ int piece_off(int row, int c) {
  const int line = D == 128 ? row : row >> 1, at = D == 128 ? c : (row & 1) * 4 + c;
  return line * 128 + ((at ^ (line & 7)) << 4);
}

template <int D, int NG, bool PAGES16>
__global__ void __launch_bounds__(THREADS) attention_q8_decode_kernel(const DecArgs a) {
  pdl_launch_dependents();
  using ST = Stage<D>;
  constexpr int KS = D / 16, CPR = D / 16;                       // k-steps of a score; 16-byte pieces of a row
  constexpr int LPT = TILE * CPR / 32;                           // pieces a lane fetches of a tile
  extern __shared__ __align__(128) unsigned char smem[];
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int G = a.H / a.KVH, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  if (!a.early) pdl_wait();
  const int seq_len = a.seq_lens[b], row_q = a.q_start[b];
  const int lo = a.window > 0 ? max(0, seq_len - a.window) : 0;
  const int tile_first = lo / TILE, total = seq_len > 0 ? (seq_len - 1) / TILE - tile_first + 1 : 0;
  const int shares = a.nsplit * WARPS, share = split * WARPS + warp;
  const int my_first = tile_first + (int)((long long)total * share / shares);
  const int n_tiles = tile_first + (int)((long long)total * (share + 1) / shares) - my_first;

  unsigned char* ring = smem + warp * ST::WARP_BYTES;
  const int* table = a.block_tables + (size_t)b * a.table_width;
  // The cache row of key (my_first + i) * TILE + lane, or -1 outside the visible range; asked for i = 0, 1, 2, ...  Table entries take longer than
  // a tile's work while the memory is busy: of pages of a multiple of 16 a lane holds the entry of 16 keys, 512 keys in all, and the
  // next 512 are on their way; of others a key's, one tile ahead.
  int pg = -1, in_page = 0, pg_next = -1, in_next = 0;
  auto fetch_pages = [&](int block) {
    const int j = (my_first + block * 16) * TILE + lane * 16, lp = j / a.page;
    in_next = j - lp * a.page;
    pg_next = (j < seq_len && j + 16 > lo && lp < a.table_width) ? table[lp] : -1;
  };
  auto row_of = [&](int i) {
    const int j = (my_first + i) * TILE + lane;
    const bool seen = i < n_tiles && j >= lo && j < seq_len;
    if (PAGES16) {
      if (i % 16 == 0) {
        pg = pg_next;
        in_page = in_next;
        fetch_pages(i / 16 + 1);
      }
      const int p = __shfl_sync(0xffffffffu, pg, i % 16 * 2 + (lane >> 4)), in = __shfl_sync(0xffffffffu, in_page, i % 16 * 2 + (lane >> 4));
      return seen && p >= 0 ? (p * a.KVH + kvh) * a.page + in + (lane & 15) : -1;
    }
    const int lp = j / a.page;
    return seen && lp < a.table_width ? (table[lp] * a.KVH + kvh) * a.page + (j - lp * a.page) : -1;
  };
  if (PAGES16) fetch_pages(0);
  auto fetch = [&](int i, int row) {                             // this lane's key's row; i < n_tiles
    unsigned char* st = ring + (i % STAGES) * ST::BYTES;
    const int c16 = lane % CPR;
#pragma unroll
    for (int u = 0; u < LPT; ++u) {
      const int key = lane / CPR + u * (32 / CPR);
      const int r = __shfl_sync(0xffffffffu, row, key);
      const size_t off = (size_t)(r < 0 ? 0 : r) * D + c16 * 16;
      const int at = piece_off<D>(key, c16);
      cp_async_16(st + at, a.cache[0] + off, r >= 0);
      cp_async_16(st + ST::TILE_BYTES + at, a.cache[1] + off, r >= 0);
    }
    float* sc = reinterpret_cast<float*>(st + 2 * ST::TILE_BYTES);
    const int pk = row < 0 ? 0 : row / a.page;                   // page * KVH + kv head
    cp_async_4(sc + lane, a.scales[0] + pk, row >= 0);
    cp_async_4(sc + TILE + lane, a.scales[1] + pk, row >= 0);
  };

  int issued = 0;
  if (a.early) {
    // Rows before the page that takes the new token were written by earlier steps: fetched while the kernels before still run.
    // (That page's scale may still grow, and its rows move with it.)
    const int settled = (seq_len - 1) / a.page * a.page;
    while (issued < min(n_tiles, STAGES - 1) && (my_first + issued + 1) * TILE <= settled) {
      fetch(issued, row_of(issued));
      cp_async_commit();
      ++issued;
    }
    pdl_wait();
  }
  for (; issued < STAGES - 1; ++issued) {
    if (issued < n_tiles) fetch(issued, row_of(issued));
    cp_async_commit();
  }
  int next_row = row_of(STAGES - 1);

  // queries: head g of the group (and g + 8), columns in the order of the keys' bytes
  unsigned qf[NG][KS][2];
  float factor[NG][2];                                           // of the heads that are this lane's columns: 2c, 2c + 1
#pragma unroll
  for (int ng = 0; ng < NG; ++ng) {
    const int head = ng * 8 + g;
    const bf16* src = a.q + (size_t)row_q * a.q_ts + (size_t)(kvh * G + min(head, G - 1)) * D + 4 * c;
    uint2 raw[KS];
    float amax = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      raw[ks] = head < G && n_tiles > 0 ? *reinterpret_cast<const uint2*>(src + ks * 16) : make_uint2(0u, 0u);
      const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].x));
      const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].y));
      amax = fmaxf(fmaxf(fmaxf(abs_or_inf(x.x), abs_or_inf(x.y)), fmaxf(abs_or_inf(y.x), abs_or_inf(y.y))), amax);
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    float f;
    const float to_half = query_to_half(amax, a.scale * LOG2E_Q8, f);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].x));
      const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].y));
      qf[ng][ks][0] = pack_half(x.x * to_half, x.y * to_half);
      qf[ng][ks][1] = pack_half(y.x * to_half, y.y * to_half);
    }
    factor[ng][0] = __shfl_sync(0xffffffffu, f, 8 * c);
    factor[ng][1] = __shfl_sync(0xffffffffu, f, 8 * c + 4);
  }

  float o[NG][KS][4];
  float m[NG][2], l[NG][2];                                      // per head of this lane's columns; l of this lane's keys alone
#pragma unroll
  for (int ng = 0; ng < NG; ++ng) {
#pragma unroll
    for (int t = 0; t < KS; ++t) o[ng][t][0] = o[ng][t][1] = o[ng][t][2] = o[ng][t][3] = 0.f;
    m[ng][0] = m[ng][1] = -INFINITY;
    l[ng][0] = l[ng][1] = 0.f;
  }
  const int mat = lane >> 3, r8 = lane & 7;
  for (int i = 0; i < n_tiles; ++i) {
    cp_async_wait<STAGES - 2>();
    __syncwarp();                                                // every lane's copies of tile i are in, and tile i - 1 is read
    if (i + STAGES - 1 < n_tiles) fetch(i + STAGES - 1, next_row);
    cp_async_commit();
    next_row = row_of(i + STAGES);
    const unsigned char* ks_ = ring + (i % STAGES) * ST::BYTES;
    const unsigned char* vs_ = ks_ + ST::TILE_BYTES;
    const float* sc = reinterpret_cast<const float*>(ks_ + 2 * ST::TILE_BYTES);
    const int j0 = (my_first + i) * TILE;
    const bool edge = j0 < lo || j0 + TILE > seq_len;
    // scores [32 keys x 8 heads]: rows g and g + 8 of two tiles of 16 keys, columns 2c and 2c + 1
    float s[NG][2][4];
#pragma unroll
    for (int ng = 0; ng < NG; ++ng)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) s[ng][mt][0] = s[ng][mt][1] = s[ng][mt][2] = s[ng][mt][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ks += 2)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        unsigned w0, w1, w2, w3, x0, x1, x2, x3;
        ldmatrix_x4(w0, w1, w2, w3, ks_ + piece_off<D>(mt * 16 + (mat & 1) * 8 + r8, ks + (mat >> 1)));
        halves_of(w0, x0, x2);
        halves_of(w1, x1, x3);
#pragma unroll
        for (int ng = 0; ng < NG; ++ng) mma_f16(s[ng][mt], x0, x1, x2, x3, qf[ng][ks][0], qf[ng][ks][1]);
        halves_of(w2, x0, x2);
        halves_of(w3, x1, x3);
#pragma unroll
        for (int ng = 0; ng < NG; ++ng) mma_f16(s[ng][mt], x0, x1, x2, x3, qf[ng][ks + 1][0], qf[ng][ks + 1][1]);
      }
    // t = score + log2 of the value's scale; online maximum per head
    float kf[2][2], back[2][2], lift[2][2];                      // [tile of 16][row g or g + 8]
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = mt * 16 + h * 8 + g;
        const float kscale = sc[key], vscale = sc[TILE + key];
        kf[mt][h] = vscale != vscale ? vscale : kscale;
        back[mt][h] = inverse_scale(vscale);
        lift[mt][h] = (float)((int)(__float_as_uint(vscale) >> 23) - 127);
      }
#pragma unroll
    for (int ng = 0; ng < NG; ++ng) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = e >> 1;
          float t = fmaf(s[ng][mt][e] * kf[mt][h], factor[ng][e & 1], lift[mt][h]);
          if (edge) {
            const int j = j0 + mt * 16 + h * 8 + g;
            t = j >= lo && j < seq_len ? t : -INFINITY;
          }
          s[ng][mt][e] = t;
          mx[e & 1] = fmaxf(mx[e & 1], t);
        }
      float corr[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 4));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 8));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 16));
        const float now = fmaxf(m[ng][e], mx[e]);                // finite, unless all that is seen is NaN (then so are the sums)
        corr[e] = ex2_q8(m[ng][e] - now);
        m[ng][e] = now;
        l[ng][e] *= corr[e];
      }
      unsigned pf[2][2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = ex2_q8(s[ng][mt][e] - m[ng][e & 1]);
          s[ng][mt][e] = p;
          l[ng][e & 1] = fmaf(p, back[mt][e >> 1], l[ng][e & 1]);
        }
        pf[mt][0] = transpose8x8(pack_half(s[ng][mt][0], s[ng][mt][1]));
        pf[mt][1] = transpose8x8(pack_half(s[ng][mt][2], s[ng][mt][3]));
      }
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        o[ng][t][0] *= corr[0];
        o[ng][t][1] *= corr[1];
        o[ng][t][2] *= corr[0];
        o[ng][t][3] *= corr[1];
      }
      s[ng][0][0] = __uint_as_float(pf[0][0]);
      s[ng][0][1] = __uint_as_float(pf[0][1]);
      s[ng][1][0] = __uint_as_float(pf[1][0]);
      s[ng][1][1] = __uint_as_float(pf[1][1]);
    }
    // outputs [D x 8 heads] += values^T [D x 32 keys] weights^T [32 keys x 8 heads]; row g of a tile of 16 columns is column 2g, row
    // g + 8 column 2g + 1
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int t = 0; t < KS; t += 2) {
        unsigned w0, w1, w2, w3, x0, x1, x2, x3;
        ldmatrix_x4_trans(w0, w1, w2, w3, vs_ + piece_off<D>(mt * 16 + (mat & 1) * 8 + r8, t + (mat >> 1)));
        halves_of(__byte_perm(w0, 0, 0x3120), x0, x1);
        halves_of(__byte_perm(w1, 0, 0x3120), x2, x3);
#pragma unroll
        for (int ng = 0; ng < NG; ++ng)
          mma_f16(o[ng][t], x0, x1, x2, x3, __float_as_uint(s[ng][mt][0]), __float_as_uint(s[ng][mt][1]));
        halves_of(__byte_perm(w2, 0, 0x3120), x0, x1);
        halves_of(__byte_perm(w3, 0, 0x3120), x2, x3);
#pragma unroll
        for (int ng = 0; ng < NG; ++ng)
          mma_f16(o[ng][t + 1], x0, x1, x2, x3, __float_as_uint(s[ng][mt][0]), __float_as_uint(s[ng][mt][1]));
      }
  }
  cp_async_wait<0>();
  __syncthreads();                                               // the rings are free: the warps' sums go over them

  constexpr int O_ROW = ST::O_ROW;
  float* o_s = reinterpret_cast<float*>(smem);                   // [WARPS][G][O_ROW]
  float* m_s = o_s + WARPS * G * O_ROW;                          // [WARPS][G]
  float* l_s = m_s + WARPS * G;                                  // [WARPS][G]
  float* M_s = l_s + WARPS * G;                                  // [G]: the block's
  float* L_s = M_s + G;
#pragma unroll
  for (int ng = 0; ng < NG; ++ng)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int head = ng * 8 + 2 * c + e;
      float sum = l[ng][e];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (head < G) {
        if (g == 0) {
          m_s[warp * G + head] = m[ng][e];
          l_s[warp * G + head] = sum;
        }
        float* dst = o_s + (size_t)(warp * G + head) * O_ROW + 2 * g;
#pragma unroll
        for (int t = 0; t < KS; ++t) *reinterpret_cast<float2*>(dst + t * 16) = make_float2(o[ng][t][e], o[ng][t][2 + e]);
      }
    }
  __syncthreads();
  // weight of a part: 2^(m - M); a part without keys (m = -inf, l = 0) has none, one whose keys are all NaN keeps that
  auto weight = [](float m1, float l1, float M) { return m1 == -INFINITY ? l1 : ex2_q8(m1 - M); };
  if ((int)threadIdx.x < G) {
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, m_s[w * G + threadIdx.x]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float l1 = l_s[w * G + threadIdx.x], f = weight(m_s[w * G + threadIdx.x], l1, M);
      L = fmaf(l1, f, L);
      m_s[w * G + threadIdx.x] = f;
    }
    M_s[threadIdx.x] = M;
    L_s[threadIdx.x] = L;
  }
  __syncthreads();
  const bool whole = a.nsplit == 1;
  for (int idx = threadIdx.x; idx < G * (D / 4); idx += THREADS) {
    const int h = idx / (D / 4), d = (idx % (D / 4)) * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = m_s[w * G + h];
      const float4 x = *reinterpret_cast<const float4*>(o_s + (size_t)(w * G + h) * O_ROW + d);
      acc.x = fmaf(x.x, f, acc.x);
      acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z);
      acc.w = fmaf(x.w, f, acc.w);
    }
    if (whole) {
      const float L = L_s[h], inv = L > 0.f ? 1.f / L : L;       // nothing seen: 0
      bf16* dst = a.out + (size_t)row_q * a.o_ts + (size_t)(kvh * G + h) * D + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
    } else if (a.cluster) {
      *reinterpret_cast<float4*>(o_s + (size_t)h * O_ROW + d) = acc;      // over the first warp's, which this thread alone reads here
    } else {
      const size_t at = ((size_t)(b * a.KVH + kvh) * a.nsplit + split) * G + h;
      *reinterpret_cast<float4*>(a.part + at * D + d) = acc;
      if (d == 0)
        *reinterpret_cast<float2*>(a.part + (size_t)a.B * a.KVH * a.nsplit * G * D + at * 2) = make_float2(M_s[h], L_s[h]);
    }
  }
  if (whole || !a.cluster) return;
  // Block `split` finishes the pieces split, split + nsplit, ... out of its peers' shared memory, in split order.
  cluster_sync_all();
  for (int piece = split + a.nsplit * (int)threadIdx.x; piece < G * (D / 4); piece += a.nsplit * THREADS) {
    const int h = piece / (D / 4), d = (piece % (D / 4)) * 4;
    float m1[8], l1[8];
    float4 x[8];
    float M = -INFINITY;
#pragma unroll
    for (int s2 = 0; s2 < 8; ++s2)
      if (s2 < a.nsplit) {
        m1[s2] = ld_peer_f32(peer_shared(M_s + h, s2));
        l1[s2] = ld_peer_f32(peer_shared(L_s + h, s2));
        x[s2] = ld_peer_v4(peer_shared(o_s + (size_t)h * O_ROW + d, s2));
        M = fmaxf(M, m1[s2]);
      }
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s2 = 0; s2 < 8; ++s2)
      if (s2 < a.nsplit) {
        const float f = weight(m1[s2], l1[s2], M);
        L = fmaf(l1[s2], f, L);
        acc.x = fmaf(x[s2].x, f, acc.x);
        acc.y = fmaf(x[s2].y, f, acc.y);
        acc.z = fmaf(x[s2].z, f, acc.z);
        acc.w = fmaf(x[s2].w, f, acc.w);
      }
    const float inv = L > 0.f ? 1.f / L : L;
    bf16* dst = a.out + (size_t)row_q * a.o_ts + (size_t)(kvh * G + h) * D + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  }
  cluster_sync_all();                                            // no block leaves while a peer still reads it
}

// The splits' sums out of scratch: one block a (kv head, request) and head of its group, a thread four columns, split order.
template <int D>
__global__ void __launch_bounds__(D / 4 * 4) attention_q8_merge_kernel(const DecArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int COLS = D / 4, PARTS = 4;                         // four threads a column cut the splits among themselves
  __shared__ float4 acc_s[PARTS][COLS];
  __shared__ float L_s[PARTS];
  const int h = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, G = a.H / a.KVH;
  const int col = threadIdx.x % COLS, part = threadIdx.x / COLS;
  const size_t first = (size_t)(b * a.KVH + kvh) * a.nsplit;
  const float* ml = a.part + (size_t)a.B * a.KVH * a.nsplit * G * D;
  float M = -INFINITY;
  for (int s = 0; s < a.nsplit; ++s) M = fmaxf(M, ml[((first + s) * G + h) * 2]);
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = part; s < a.nsplit; s += PARTS) {
    const float2 x = *reinterpret_cast<const float2*>(ml + ((first + s) * G + h) * 2);
    const float4 y = *reinterpret_cast<const float4*>(a.part + ((first + s) * G + h) * D + col * 4);
    const float f = x.x == -INFINITY ? x.y : ex2_q8(x.x - M);
    L = fmaf(x.y, f, L);
    acc.x = fmaf(y.x, f, acc.x);
    acc.y = fmaf(y.y, f, acc.y);
    acc.z = fmaf(y.z, f, acc.z);
    acc.w = fmaf(y.w, f, acc.w);
  }
  acc_s[part][col] = acc;
  if (col == 0) L_s[part] = L;
  __syncthreads();
  if (part != 0) return;
  for (int p = 1; p < PARTS; ++p) {
    const float4 y = acc_s[p][col];
    acc.x += y.x;
    acc.y += y.y;
    acc.z += y.z;
    acc.w += y.w;
    L += L_s[p];
  }
  const float inv = L > 0.f ? 1.f / L : L;
  bf16* dst = a.out + (size_t)a.q_start[b] * a.o_ts + (size_t)(kvh * G + h) * D + col * 4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

template <int D, int NG, bool PAGES16>
int prepare_kernel() {
  static const int slots = [] {
    if (cudaFuncSetAttribute(attention_q8_decode_kernel<D, NG, PAGES16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Stage<D>::SMEM) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attention_q8_decode_kernel<D, NG, PAGES16>, THREADS, Stage<D>::SMEM) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    return n;
  }();
  return slots;
}

// How many clusters of n blocks the chip holds at once.
template <int D, int NG, bool PAGES16>
int clusters_that_fit(int n) {
  static int known[9];
  int& k = known[n];
  if (k == 0) {
    k = -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n, 1, 1);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Stage<D>::SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)n;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, attention_q8_decode_kernel<D, NG, PAGES16>, &cfg) == cudaSuccess && clusters >= 1) k = clusters;
    cudaGetLastError();                                          // a refusal is an answer, not an error
  }
  return k;
}

template <int D, int NG, bool PAGES16>
int launch(const DecArgs& a, cudaStream_t s) {
  if (prepare_kernel<D, NG, PAGES16>() == 0) TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_decode: the device does not hold a block");
  cudaError_t e = ts_launch_cluster(attention_q8_decode_kernel<D, NG, PAGES16>, dim3(a.cluster ? a.nsplit : 1, 1, 1), dim3(a.nsplit, a.KVH, a.B),
                                    dim3(THREADS), Stage<D>::SMEM, s, a);
  if (e != cudaSuccess) TS_REFUSE((int)e, "ts_attention_q8_decode: %s", cudaGetErrorString(e));
  if (a.nsplit > 1 && !a.cluster) {
    e = ts_launch(attention_q8_merge_kernel<D>, dim3(a.H / a.KVH, a.KVH, a.B), dim3(D), 0, s, a);
    if (e != cudaSuccess) TS_REFUSE((int)e, "ts_attention_q8_decode: %s", cudaGetErrorString(e));
  }
  TS_LAUNCH_CHECK();
}

}  // namespace

static bool decode_takes(int H, int KVH, int D) { return KVH > 0 && H % KVH == 0 && H / KVH <= 16 && (D == 64 || D == 128); }

// Blocks of the kernel that an SM holds at once, for groups of G heads of D.
TS_API int ts_attention_q8_decode_blocks_per_sm(int G, int D) {
  if (!decode_takes(G, 1, D)) return 0;
  if (D == 64) return G <= 8 ? prepare_kernel<64, 1, true>() : prepare_kernel<64, 2, true>();
  return G <= 8 ? prepare_kernel<128, 1, true>() : prepare_kernel<128, 2, true>();
}

// Clusters of n blocks (2 to 8) that the device holds at once, whether or not they are switched on; 0: none.
TS_API int ts_attention_q8_decode_clusters(int G, int D, int n) {
  if (n < 2 || n > 8 || ts_attention_q8_decode_blocks_per_sm(G, D) == 0) return 0;
  const int k = D == 64 ? (G <= 8 ? clusters_that_fit<64, 1, true>(n) : clusters_that_fit<64, 2, true>(n))
                        : (G <= 8 ? clusters_that_fit<128, 1, true>(n) : clusters_that_fit<128, 2, true>(n));
  return k < 0 ? 0 : k;
}

// One query token per request (rows q_start[b]).  nsplit: blocks that cut the keys of a (request, kv head) among themselves; cluster: as one
// cluster (2 to 8 of them), else with B * H * nsplit * (D + 2) floats of scratch.  early: index arrays and cache rows before
// each request's last page are in place already and are read before the wait for the kernels before.
TS_API int ts_attention_q8_decode(const void* record, void* stream) {
  const AttendCall& c = *(const AttendCall*)record;
  const int B = c.B, H = c.H, KVH = c.KVH, D = c.D, page = c.page, num_pages = c.num_pages, nsplit = c.nsplit, cluster = c.cluster;
  const long long o_ts = c.o_ts, q_ts = c.q_ts;
  const void *const k_cache = c.k_cache, *const v_cache = c.v_cache, *const q = c.q;
  void* const out = c.out;
  float* const scratch = c.scratch;
  if (B <= 0) return 0;
  if (!decode_takes(H, KVH, D) || page <= 0)
    TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_decode: H=%d KVH=%d D=%d page=%d is not taken by this kernel", H, KVH, D, page);
  if (nsplit < 1 || nsplit > 128 || (cluster && (nsplit < 2 || nsplit > 8)) || (nsplit > 1 && !cluster && scratch == nullptr))
    TS_REFUSE(TS_ERR_LIMIT, "ts_attention_q8_decode: %d splits%s", nsplit, cluster ? " as a cluster" : "");
  if (cluster && !ts_clusters_enabled()) TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_decode: thread-block clusters are switched off");
  if (B > 65535 || KVH > 65535) TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_decode: %d requests / %d kv heads", B, KVH);
  if ((((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)scratch) & 15) != 0 || (((uintptr_t)q | (uintptr_t)out) & 7) != 0 ||
      (q_ts & 3) != 0 || (o_ts & 3) != 0)
    TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_decode: pages on 16 bytes, rows of queries and outputs on 8");
  if ((long long)num_pages * KVH * page > 0x7fffffffLL) TS_REFUSE(TS_ERR_UNSUPPORTED, "ts_attention_q8_decode: a cache of more than 2^31 rows");
  DecArgs a = {(bf16*)out, o_ts, (const bf16*)q, q_ts, {(const unsigned char*)k_cache, (const unsigned char*)v_cache},
               {c.k_scale, c.v_scale}, c.block_tables, c.q_start, c.seq_lens, scratch, B, c.table_width, H, KVH, page, c.scale, c.window, nsplit,
               cluster, c.early};
  cudaStream_t s = (cudaStream_t)stream;
  const int G = H / KVH;
  if (page % 16 == 0) {
    if (D == 64) return G <= 8 ? launch<64, 1, true>(a, s) : launch<64, 2, true>(a, s);
    return G <= 8 ? launch<128, 1, true>(a, s) : launch<128, 2, true>(a, s);
  }
  if (D == 64) return G <= 8 ? launch<64, 1, false>(a, s) : launch<64, 2, false>(a, s);
  return G <= 8 ? launch<128, 1, false>(a, s) : launch<128, 2, false>(a, s);
}
