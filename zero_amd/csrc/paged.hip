// Serving operators over a paged key / value cache: append with rotation, attention of new tokens.
//
// The cache of one layer is two bf16 arrays [n_pages][page_size][Hkv * hd] (keys after rotation, values); a sequence
// owns the pages its row of the page table names, so its cached row r is row r % page_size of page table[r / page_size].
// The layout is the token-major one of the contiguous caches (zk_attn_decode): the new rows of a token are one store,
// and a contiguous cache [B][rows][Hkv * hd] is the special case of one page per sequence.
// Every index that comes from device memory (slots, positions, page numbers, lengths) is checked in the kernel against
// the sizes the host passed: nothing is read or written outside the arrays whatever the tables hold.
#include "attn_common.h"
#include "../../include/zero_hip.h"

using namespace zkattn;

namespace {

constexpr float kLog2e = LOG2E;
// The softmax is relative to a maximum that may lag the true one by this power of two: outputs and sums are rescaled only
// when a score passes it (64 multiplies a piece otherwise), and neither fp32 sums nor bf16 probabilities lose anything to a
// common factor of up to 2^8.
constexpr float kSlack = 8.0f;

// =========================================================================================
// append, bound by memory (8191 tokens of 32 + 2 * 8 heads of 128: 206 MB in 33.7 us, 6.1 TB/s): one workgroup per token, a
// unit of work is 16 values of a head (two 16-byte chunks) that turn by 8 angles.
// half layout: chunks p and p + rot/16 of the head; interleaved: chunks 2p and 2p + 1 (pairs inside a chunk); chunks
// past rot, and the values, are copied.
// =========================================================================================
template <int HD>
__global__ __launch_bounds__(256) void kv_append_paged_kernel(const bf16_t* qkv, const float* cos_t, const float* sin_t,
                                                              bf16_t* q_out, bf16_t* k_cache, bf16_t* v_cache,
                                                              const int* positions, const int* slots, int Hq, int Hkv,
                                                              int rot, int table_rows, long long ldqkv, long long ldq,
                                                              long long cache_rows, int interleaved) {
  constexpr int UPH = HD / 16;                      // units per head
  const int t = blockIdx.x;
  const int pos = positions[t], slot = slots[t];
  const bool live = pos >= 0 && pos < table_rows;   // otherwise a padding token: q row of zeros, nothing appended
  const bool keep = live && slot >= 0 && slot < cache_rows;
  const int half = rot >> 1, kvw = Hkv * HD;
  const bf16_t* row = qkv + (size_t)t * ldqkv;
  const int units = (Hq + 2 * Hkv) * UPH;
  for (int i = threadIdx.x; i < units; i += 256) {
    const int head = i / UPH, p = i % UPH;
    if (head >= Hq && !keep) continue;
    const bool turned = head < Hq + Hkv && p < (rot >> 4);
    int c0 = 2 * p, c1 = 2 * p + 1;
    if (turned && !interleaved) { c0 = p; c1 = p + (rot >> 4); }
    u32x4 a = *reinterpret_cast<const u32x4*>(row + head * HD + c0 * 8);
    u32x4 b = *reinterpret_cast<const u32x4*>(row + head * HD + c1 * 8);
    if (turned && live) {
      const float* cp = cos_t + (size_t)pos * half + p * 8;
      const float* sp = sin_t + (size_t)pos * half + p * 8;
      float cs[8], sn[8];
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        *reinterpret_cast<f32x4*>(cs + e) = *reinterpret_cast<const f32x4*>(cp + e);
        *reinterpret_cast<f32x4*>(sn + e) = *reinterpret_cast<const f32x4*>(sp + e);
      }
      if (interleaved) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x, y;
          rope_pair(lo_bf(a[e]), hi_bf(a[e]), cs[e], sn[e], x, y);
          a[e] = pack2bf(x, y);
          rope_pair(lo_bf(b[e]), hi_bf(b[e]), cs[4 + e], sn[4 + e], x, y);
          b[e] = pack2bf(x, y);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x0, y0, x1, y1;
          rope_pair(lo_bf(a[e]), lo_bf(b[e]), cs[2 * e], sn[2 * e], x0, y0);
          rope_pair(hi_bf(a[e]), hi_bf(b[e]), cs[2 * e + 1], sn[2 * e + 1], x1, y1);
          a[e] = pack2bf(x0, x1);
          b[e] = pack2bf(y0, y1);
        }
      }
    }
    bf16_t* dst;
    if (head < Hq) {
      if (!live) { a = u32x4{0u, 0u, 0u, 0u}; b = a; }
      dst = q_out + (size_t)t * ldq + head * HD;
    } else if (head < Hq + Hkv) {
      dst = k_cache + (size_t)slot * kvw + (head - Hq) * HD;
    } else {
      dst = v_cache + (size_t)slot * kvw + (head - Hq - Hkv) * HD;
    }
    *reinterpret_cast<u32x4*>(dst + c0 * 8) = a;
    *reinterpret_cast<u32x4*>(dst + c1 * 8) = b;
  }
}

struct PagedArgs {
  const bf16_t *q, *k, *v;
  bf16_t* out;
  const int *table, *ctx, *cu;
  const unsigned long long* mask;
  // shares' un-normalised outputs and (maximum, sum): [T * Hq][splits][HD], [..][2] (stream kernel) or
  // [workgroup][128 rows][HD], [..][2] with the layout in `shares` (tile kernel); null: no sequence is shared out
  float *part_o, *part_ml;
  int* shares;
  int T, B, max_q, Hq, Hkv, page_size, n_pages, table_cols, ld_table, mask_words;
  int splits, split_keys;
  unsigned page_mul, page_shift;   // key / page_size = key * page_mul >> page_shift for every key < 2^31
  long long ldq, ldo;
  float scale;
};

constexpr int kMaxRows = 1 << 30;

// the larger of a value and that of the lane 16 / 32 away, without LDS (v_permlane{16,32}_swap of a value with itself
// leaves the even halves in one register and the odd ones in the other)
__device__ __forceinline__ float max_over16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_over32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// one sequence's share of the call
struct Seq {
  int q0, n, len;               // first row of q, new tokens, cached rows
  int first;                    // cached rows before the new tokens (as the lengths say: negative if they do not fit)
  int rows;                     // of a kv head: computed tokens times the heads that share it
  __device__ __forceinline__ Seq(const PagedArgs& a, int b) {
    q0 = min(max(a.cu[b], 0), a.T);
    n = min(max(a.cu[b + 1], q0), a.T) - q0;
    const int c = min(max(a.ctx[b], 0), kMaxRows);  // and T < kMaxRows: differences of the two fit 32 bits
    len = (int)min((long long)c, (long long)a.table_cols * a.page_size);
    first = c - n;
    rows = min(n, a.max_q) * (a.Hq / a.Hkv);
  }
};

// the sequence that row t of q belongs to if it belongs to one, by the ends at or before it (whole waves, one t a wave)
__device__ __forceinline__ int seq_of(const PagedArgs& a, int t) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) n += __popcll(__ballot(b0 + lane < a.B && a.cu[min(b0 + lane, a.B - 1) + 1] <= t));
  return min(n, a.B - 1);
}

// which of the 32 keys from `base` on new token i (row q0 + i of q) may see, as bits; the cache's end is not looked at
__device__ __forceinline__ unsigned seen_bits(const PagedArgs& a, const Seq& s, int i, int base) {
  const int j0 = base - s.first;                    // key `base` is new token j0 (negative: a row before them)
  if (!a.mask) {                                    // keys up to the token's own
    const int c = i - j0 + 1;
    return c >= 32 ? ~0u : c <= 0 ? 0u : (1u << c) - 1u;
  }
  if (j0 <= -32) return ~0u;
  const unsigned long long* m = a.mask + (size_t)(s.q0 + i) * a.mask_words;
  if (j0 < 0) return (unsigned)(m[0] << -j0) | ((1u << -j0) - 1u);
  const int w = j0 >> 6, sh = j0 & 63;
  unsigned long long x = w < a.mask_words ? m[w] >> sh : 0ull;
  if (sh > 32 && w + 1 < a.mask_words) x |= m[w + 1] << (64 - sh);
  return (unsigned)x;
}

// flat cache row of key `key` of sequence b, or -1: past `end`, or on a page that does not exist
__device__ __forceinline__ int cache_row(const PagedArgs& a, int b, int key, int end) {
  if (key >= end) return -1;
  const unsigned at = (unsigned)(((unsigned long long)(unsigned)key * a.page_mul) >> a.page_shift);
  const unsigned pg = (unsigned)a.table[(size_t)b * a.ld_table + at];
  return pg < (unsigned)a.n_pages ? (int)(pg * (unsigned)a.page_size + ((unsigned)key - at * (unsigned)a.page_size)) : -1;
}

// Shares of the tile kernel's work, from the lengths themselves (the host knows bounds only; shares cut by the largest
// length left half of the CUs idle on a ragged batch).  A share is `q` 64-key tiles of one (sequence, kv head, 128-row
// tile); q is the cut of the longest sequence into 1 .. 64 that minimises rounds * (q + 4), 4 tiles being what a share costs
// beside its own (prologue, stores, merge), with the workgroups that the GPU holds at once as a round.  Each wave works
// it out for itself, lane i trying the cut into i + 1.  Workgroup ids run over sequences, row tiles, shares, kv heads:
// with 8 kv heads the row tiles of a share are on one XCD (ids equal modulo 8) and its L2 serves all but the first.
template <int HD>
constexpr int kTileSlots = HD == 64 ? 768 : 512;    // three / two workgroups a CU
struct Shares {
  int q, b = -1, tile = 0, unit = 0, units = 0;     // unit = share * Hkv + kv head, of `units`; b < 0: no work
  __device__ __forceinline__ static void of(const PagedArgs& a, int b, int& tiles, int& len) {
    tiles = len = 0;
    if (b >= a.B) return;
    const Seq s(a, b);
    tiles = (s.rows + 127) >> 7;
    len = max((s.len + 63) >> 6, 1);
  }
  __device__ __forceinline__ Shares(const PagedArgs& a, int slots, int id) {
    const int lane = threadIdx.x & 63;
    int tiles, len, all = 0, longest = 1;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      of(a, b0 + lane, tiles, len);
      all += tiles;
      longest = max(longest, tiles ? len : 1);      // (B <= 64: the lanes keep their sequence's)
    }
    all = __builtin_amdgcn_readlane(wave_upto(all), 63) * a.Hkv;
    longest = wave_top(longest);
    q = longest;
    if (a.part_o && longest > 4 && all < 2 * slots) {
      const int mine = (longest + lane) / (lane + 1);
      const float inv = 1.0f / (float)mine;
      int n = 0;
      for (int b0 = 0; b0 < a.B; b0 += 64) {
        if (a.B > 64) of(a, b0 + lane, tiles, len);
        for (int j = 0; j < min(64, a.B - b0); ++j)
          n += __builtin_amdgcn_readlane(tiles, j) * (int)(((float)(__builtin_amdgcn_readlane(len, j) + mine) - 0.5f) * inv);
      }
      n *= a.Hkv;
      int cost = (n + slots - 1) / slots * (mine + 4);
      if (n > 2 * slots && lane) cost = 0x1FFFFFF;
      const int best = -wave_top(-((min(cost, 0x1FFFFFF) << 6) | lane));
      q = (longest + (best & 63)) / ((best & 63) + 1);
    }
    for (;;) {
      b = -1;
      int before = 0;
      for (int b0 = 0; b0 < a.B; b0 += 64) {
        if (a.B > 64) of(a, b0 + lane, tiles, len);
        const int u = a.Hkv * ((len + q - 1) / q), n = tiles * u;
        const int upto = wave_upto(n);
        const int start = before + upto - n;
        if (id == 0 && threadIdx.x < 64 && a.part_o && b0 + lane < a.B) a.shares[1 + b0 + lane] = start;
        const unsigned long long hit = __ballot(id >= start && id < start + n);
        if (hit) {
          const int at = __ffsll(hit) - 1;
          b = b0 + at;
          units = __builtin_amdgcn_readlane(u, at);
          unit = id - __builtin_amdgcn_readlane(start, at);
          tile = unit / units;
          unit -= tile * units;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
      }
      if (q == longest || before <= 2 * slots) break;
      q = longest;                                  // (the choice above counts in fp32)
    }
    if (id == 0 && threadIdx.x == 0 && a.part_o) a.shares[0] = q == longest ? 0 : q;
    q = __builtin_amdgcn_readfirstlane(q);          // (all of these are the same in the workgroup)
    b = __builtin_amdgcn_readfirstlane(b);
    tile = __builtin_amdgcn_readfirstlane(tile);
    unit = __builtin_amdgcn_readfirstlane(unit);
    units = __builtin_amdgcn_readfirstlane(units);
  }
};

__device__ __forceinline__ bool not_finite(unsigned w) {
  return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
}

// =========================================================================================
// attention of few rows.  The q rows of a group of Hq / Hkv heads read the same keys, so a workgroup takes all rows of one kv
// head (token i, head g of the group at row i * G + g; 16 * MT at most) over one share of a sequence's keys.  Workgroup ids
// run over sequences, shares, kv heads: neighbours are on different XCDs, so that a long sequence loads all of them.
// Its W waves take 32-key pieces in turn, each with a softmax of its own (running maximum and sum in fp32, no barrier in
// the loop), merged through LDS at the end; shares of one sequence are merged by attn_paged_merge_kernel.
// Products: 16x16x32 MFMAs.  S^T[key][row] = K Q^T, K fragments straight from memory to registers (16 rows x 64 bytes per
// load); a lane then owns 8 keys of one row, which are the B operand of O^T += V^T P^T as they stand if V^T is read in
// the same key order (elements 0-3 keys 4g.., 4-7 keys 16 + 4g.. of lane group g): ds_read_b64_tr_b16 from the wave's own
// copy of V in LDS, chunk-swizzled by the row.  The next piece's rows are requested as soon as a piece's registers are free.
// Bound by memory: 48 sequences of 700 to 8192 rows (8 kv heads of 128, 633 MB) 132 us, 4.8 TB/s; one of 131071 (8 heads
// over one of 128, 67 MB) 15.7 us, 4.3 TB/s.  A short call is latency: 768 rows in 5.9 us, three dependent loads and a merge.
// =========================================================================================
template <int HD, int MT, int W>
__global__ __launch_bounds__(64 * W, W == 4 && MT == 1 && HD == 64 ? 4 : 2) void attn_paged_stream_kernel(PagedArgs a) {
  constexpr int CPR = HD / 8, KC = HD / 32, DB = HD / 16, NV = HD / 16;
  constexpr int LDO = HD + 4;                       // floats per row of the waves' exchange: 16 rows hit different banks
  constexpr int VB = 32 * HD * 2;                   // one wave's V piece
  constexpr int XB = W * 16 * LDO * 4;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[XB > W * VB ? XB : W * VB];
  __shared__ float sm[W][16 * MT], sl[W][16 * MT];
  const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = (int)blockIdx.x % a.Hkv, split = (int)blockIdx.x / a.Hkv % a.splits, b = (int)blockIdx.x / a.Hkv / a.splits;
  const Seq s(a, b);
  const int G = a.Hq / a.Hkv, rows = s.rows, kvw = a.Hkv * HD;
  const int ks = split * a.split_keys;
  if (!rows || (split > 0 && ks >= s.len)) return;
  const int ke = split == a.splits - 1 ? s.len : min(s.len, ks + a.split_keys);
  const bool alone = ks == 0 && ke == s.len;        // no other share of this sequence
  const float sc = a.scale * kLog2e;
  const bf16_t* kb = a.k + kvh * HD;
  const bf16_t* vb = a.v + kvh * HD;

  bf16x8 q[MT][KC];
  int tok[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = mt * 16 + col;
    tok[mt] = min(r, rows - 1) / G;
    const bf16_t* qp = a.q + (size_t)(s.q0 + tok[mt]) * a.ldq + (size_t)(kvh * G + min(r, rows - 1) % G) * HD + 8 * g4;
#pragma unroll
    for (int c = 0; c < KC; ++c) q[mt][c] = *reinterpret_cast<const bf16x8*>(qp + 32 * c);
  }
  f32x4 o[MT][DB];
  float m[MT], l[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -INFINITY; l[mt] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  unsigned char* vl = smem + wave * VB;
  bf16x8 kf[2][KC];
  u32x4 vr[NV];
  f32x4 sc4[MT][2];
  bf16x8 p[MT];
  auto request = [&](int r) __attribute__((always_inline)) {      // a piece's rows; lane & 31 holds key lane & 31's
#pragma unroll
    for (int kg = 0; kg < 2; ++kg) {
      const bf16_t* x = kb + (size_t)max(__shfl(r, kg * 16 + col, 64), 0) * kvw + 8 * g4;
#pragma unroll
      for (int c = 0; c < KC; ++c) kf[kg][c] = *reinterpret_cast<const bf16x8*>(x + 32 * c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int idx = i * 64 + lane;
      vr[i] = *reinterpret_cast<const u32x4*>(vb + (size_t)max(__shfl(r, idx / CPR, 64), 0) * kvw + (idx % CPR) * 8);
    }
  };
  auto scores = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int kg = 0; kg < 2; ++kg)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c) z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kg][c], q[mt][c], z, 0, 0, 0);
        sc4[mt][kg] = z;
      }
  };
  auto v_at = [&](int vrow, int ch) { return vl + vrow * (HD * 2) + ((ch ^ ((vrow & (CPR / 2 - 1)) << 1)) << 4); };
  // a value's lanes write, other lanes read: nothing may move across in the compiler either (the wave's own LDS
  // instructions are in order)
  auto lds_turn = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  };
  auto softmax = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float mx = sc4[mt][0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sc4[mt][e >> 2][e & 3]);
      mx = max_over32(max_over16(mx));
      mx *= sc;
      if (__any(mx > m[mt] + kSlack)) {
        const float mn = fmaxf(m[mt], mx), f = fast_exp2(m[mt] - (mn == -INFINITY ? 0.f : mn));
        l[mt] *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[mt][d] *= f;
        m[mt] = mn;
      }
      const float use = m[mt] == -INFINITY ? 0.f : m[mt];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = fast_exp2(__builtin_fmaf(sc4[mt][e >> 2][e & 3], sc, -use));
        l[mt] += x;
        p[mt][e] = (__bf16)x;                       // rounded to bf16 for the matrix product only
      }
    }
  };
  auto product = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const unsigned char* at = v_at(4 * g4 + (col >> 2), 2 * d + ((col & 3) >> 1)) + (col & 1) * 8;
      union { struct { short4_t lo, hi; } h; bf16x8 v; } u;
      u.h.lo = lds_read_tr16(at);
      u.h.hi = lds_read_tr16(at + 16 * (HD * 2));   // 16 rows on: the same swizzle
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[mt][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u.v, p[mt], o[mt][d], 0, 0, 0);
    }
  };

  // pieces that every row sees whole: up to the first new token in a chain, to the new tokens in a tree
  const int bulk = min(ke, s.first + (a.mask ? 0 : 1));
  int base = ks + 32 * wave;
  if (base + 32 <= bulk) {
    int row = cache_row(a, b, base + (lane & 31), bulk);
    request(row);
    int ahead = cache_row(a, b, base + 32 * W + (lane & 31), bulk);
    while (__all(row >= 0)) {
      scores();
#pragma unroll
      for (int i = 0; i < NV; ++i) *reinterpret_cast<u32x4*>(v_at((i * 64 + lane) / CPR, (i * 64 + lane) % CPR)) = vr[i];
      lds_turn();
      base += 32 * W;
      row = ahead;
      if (base + 32 <= bulk) {
        request(row);
        ahead = cache_row(a, b, base + 32 * W + (lane & 31), bulk);
      }
      softmax();
      product();
      lds_turn();
      if (base + 32 > bulk) break;
    }
  }
  // the others: the cache's end, new tokens, pages that do not exist (and what stands behind one)
  for (; base < ke; base += 32 * W) {
    const int row = cache_row(a, b, base + (lane & 31), ke);
    request(row);
    scores();
    const unsigned ok = (unsigned)__ballot(row >= 0);
    bool odd = false;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int vrow = (i * 64 + lane) / CPR;
      u32x4 x = vr[i];
      if (!((ok >> vrow) & 1)) x = u32x4{0u, 0u, 0u, 0u};      // its p is 0, and 0 x NaN is not
#pragma unroll
      for (int e = 0; e < 4; ++e) odd |= not_finite(x[e]);
      *reinterpret_cast<u32x4*>(v_at(vrow, (i * 64 + lane) % CPR)) = x;
    }
    lds_turn();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const unsigned vis = seen_bits(a, s, tok[mt], base) & ok;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!((vis >> (16 * (e >> 2) + 4 * g4 + (e & 3))) & 1)) sc4[mt][e >> 2][e & 3] = -INFINITY;
    }
    softmax();
    if (!__any(odd)) {
      product();
    } else {
      // infinities or NaN among cache rows that some tokens may not see: key by key, rows with p = 0 passed over
#pragma unroll 1
      for (int vrow = 0; vrow < 32; ++vrow) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float x = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e == 4 * (vrow >> 4) + (vrow & 3)) x = (float)p[mt][e];
          x = __shfl(x, ((vrow >> 2) & 3) * 16 + col, 64);
          if (x == 0.f) continue;
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(v_at(vrow, 2 * d + (g4 >> 1)) + (g4 & 1) * 8);
            o[mt][d][0] += x * lo_bf(w[0]); o[mt][d][1] += x * hi_bf(w[0]);
            o[mt][d][2] += x * lo_bf(w[1]); o[mt][d][3] += x * hi_bf(w[1]);
          }
        }
      }
    }
    lds_turn();
  }
  // ---- the waves' shares, in wave order
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    l[mt] += __shfl_xor(l[mt], 16, 64);
    l[mt] += __shfl_xor(l[mt], 32, 64);
    if (g4 == 0) { sm[wave][mt * 16 + col] = m[mt]; sl[wave][mt * 16 + col] = l[mt]; }
  }
  float* xo = reinterpret_cast<float*>(smem);
  constexpr int per = HD / (4 * W);                  // columns a thread writes
  const int orow = tid / (4 * W), oc = (tid % (4 * W)) * per;
  auto top = [&](int r) {
    float M = sm[0][r];
#pragma unroll
    for (int w = 1; w < W; ++w) M = fmaxf(M, sm[w][r]);
    return M;
  };
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    __syncthreads();
    {
      const int r = mt * 16 + col;
      const float M = top(r);
      const float f = M == -INFINITY ? 0.f : fast_exp2(m[mt] - M);
#pragma unroll
      for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4*>(xo + (wave * 16 + col) * LDO + d * 16 + 4 * g4) = o[mt][d] * f;
    }
    __syncthreads();
    const int r = mt * 16 + orow;
    if (r < rows) {
      const float M = top(r);
      float L = 0.f, y[per];
#pragma unroll
      for (int w = 0; w < W; ++w) L += M == -INFINITY ? 0.f : sl[w][r] * fast_exp2(sm[w][r] - M);
#pragma unroll
      for (int e = 0; e < per; ++e) {
        y[e] = 0.f;
#pragma unroll
        for (int w = 0; w < W; w += 4)
          y[e] += (xo[(16 * w + orow) * LDO + oc + e] + xo[(16 * w + 16 + orow) * LDO + oc + e]) +
                  (xo[(16 * w + 32 + orow) * LDO + oc + e] + xo[(16 * w + 48 + orow) * LDO + oc + e]);
      }
      const int t = s.q0 + r / G, h = kvh * G + r % G;
      if (alone) {
        const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);      // nothing seen: zeros; NaN stays NaN
        bf16_t* op = a.out + (size_t)t * a.ldo + (size_t)h * HD + oc;
#pragma unroll
        for (int e = 0; e < per; e += W == 4 ? 4 : 2)
          if constexpr (W == 4) {
            u32x2 w = {pack2bf(y[e] * inv, y[e + 1] * inv), pack2bf(y[e + 2] * inv, y[e + 3] * inv)};
            *reinterpret_cast<u32x2*>(op + e) = w;
          } else {
            *reinterpret_cast<unsigned*>(op + e) = pack2bf(y[e] * inv, y[e + 1] * inv);
          }
      } else {
        const size_t part = ((size_t)t * a.Hq + h) * a.splits + split;
#pragma unroll
        for (int e = 0; e < per; e += 4)            // (8 waves: no call has shares)
          if constexpr (W == 4)
            *reinterpret_cast<f32x4*>(a.part_o + part * HD + oc + e) = f32x4{y[e], y[e + 1], y[e + 2], y[e + 3]};
        if (oc == 0) { a.part_ml[part * 2] = M; a.part_ml[part * 2 + 1] = L; }
      }
    }
  }
}

// =========================================================================================
// the same for many rows (prompt chunks, large trees): a workgroup is 128 rows of one kv head, four waves of 32 rows that
// share every 64-key tile.  K and V tiles arrive by LDS-DMA (per-lane 64-bit source addresses: the rows of a paged cache),
// chunk-swizzled, two stages, one barrier per tile; S^T = K Q^T and O^T += V^T P^T in 32x32x16 MFMAs with the row on
// the lane, as in zk_attn_fwd.  Each wave's instructions bind, matrix and vector in turn: a 64-key tile takes a workgroup
// 2.5 us, of which 1.7 us stay without the matrix instructions and 2.0 us without the DMA.  2048 new tokens over 32768 rows
// (32 heads over 8 of 128, 1.06 TFLOP; 512 workgroups, one round): calls of 1046 to 1129 us from card to card, 940 to 1010
// TFLOP/s, and 1100 to 1177 us a launch in a kernel trace of nine.  2112 to 2560 tokens take 1800 us, a second round that is
// nearly empty; a whole prompt's row tiles differ in length: 2048 tokens 76 us, 8192 659 (452 and 835 TFLOP/s).  Short
// chunks are latency: a share's start, its stores and the merge cost as much as four of its tiles.
// =========================================================================================
// LDS-DMA of 16 bytes a lane to consecutive LDS from the wave-uniform `dst` on; sources per lane, or a uniform base and a
// 32-bit byte offset.  Inline asm, not the builtin: behind a builtin the compiler waits for every DMA in flight before the
// first transposed LDS read, whatever tile that reads, and so for tile t + 1 in the middle of tile t.  The loop waits by
// hand (vmcnt(0) and a barrier before a tile's first read); no register is written, m0 is used by nothing else here.
__device__ __forceinline__ void lds_dma_from(const void* dst, const void* src) {
  const unsigned m = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long)(__attribute__((address_space(3))) void*)const_cast<void*>(dst));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(m), "v"(src) : "memory");
}
__device__ __forceinline__ void lds_dma_at(const void* dst, const void* base, unsigned off) {
  const unsigned m = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long)(__attribute__((address_space(3))) void*)const_cast<void*>(dst));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m), "v"(off), "s"(base) : "memory");
}
// ONE_PAGE: page_size is a multiple of 64, so a tile lies in one page: its address is uniform and a lane's offset into it
// constant, where pages of any size cost a look-up, four exchanges and 64-bit multiplies a lane and tile.
template <int HD, bool ONE_PAGE>
__global__ __launch_bounds__(256, kTileSlots<HD> / 256) void attn_paged_tile_kernel(PagedArgs a) {
  using C = Cfg<HD>;
  constexpr int KV = 64, RB = HD * 2, TB = KV * RB, STAGE = 2 * TB, CPR = HD / 8, NQ = KV * CPR / 256;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * STAGE];
  __shared__ unsigned bad[2];
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Shares w(a, kTileSlots<HD>, (int)blockIdx.x);
  if (w.b < 0) return;
  const int b = w.b, split = __builtin_amdgcn_readfirstlane(w.unit / a.Hkv), kvh = w.unit - split * a.Hkv;
  const Seq s(a, b);
  const int G = a.Hq / a.Hkv, rows = s.rows, kvw = a.Hkv * HD, t0 = w.tile * 128;
  const int ks = split * w.q * KV, ke = min(s.len, ks + w.q * KV);
  const bool alone = w.units == a.Hkv;
  const float sc = a.scale * kLog2e;
  const int r0 = t0 + wave * 32, r = r0 + (lane & 31), rc = min(r, rows - 1), tok = rc / G;
  // keys that the workgroup / this wave needs at all, and those that every row of the workgroup sees
  const int last_wg = a.mask ? s.len : s.first + min(t0 + 127, rows - 1) / G + 1;
  const int last_wave = r0 >= rows ? 0 : a.mask ? s.len : s.first + min(r0 + 31, rows - 1) / G + 1;
  const int clear = min(ke, s.first + (a.mask ? 0 : t0 / G + 1));
  const int nt = (min(ke, max(last_wg, ks)) - ks + KV - 1) / KV;
  const bf16_t* kb = a.k + kvh * HD;
  const bf16_t* vb = a.v + kvh * HD;

  int row, next = -1;                               // cache row of key `lane` (ONE_PAGE: of the first key) of a tile
  auto look = [&](int t) __attribute__((always_inline)) { return cache_row(a, b, ks + t * KV + (ONE_PAGE ? 0 : lane), ke); };
  // A tile's DMA in 2 NQ pieces (16 bytes a lane; even: K, odd: V).  Behind the barrier they go out one between the
  // matrix instructions of each k-step: in a burst each holds its wave for 60 to 180 cycles.
  size_t from[ONE_PAGE ? 1 : NQ];
  auto aim = [&](int rr) __attribute__((always_inline)) {
    if (ONE_PAGE) {
      from[0] = (size_t)max(__builtin_amdgcn_readfirstlane(rr), 0) * kvw;
    } else {
#pragma unroll
      for (int i = 0; i < NQ; ++i) from[i] = (size_t)max(__shfl(rr, (tid + 256 * i) / CPR, 64), 0) * kvw;
    }
  };
  auto piece = [&](int t, int i2) __attribute__((always_inline)) {
    const int i = i2 >> 1, sidx = tid + 256 * i, trow = sidx / CPR, ch = (sidx % CPR) ^ swz_key<HD>(trow);
    unsigned char* dst = smem + (t & 1) * STAGE + (i2 & 1) * TB + (wave * 64 + 256 * i) * 16;
    const bf16_t* src = i2 & 1 ? vb : kb;
    if (ONE_PAGE) lds_dma_at(dst, src + from[0], (unsigned)(trow * kvw + ch * 8) * 2u);
    else lds_dma_from(dst, src + from[ONE_PAGE ? 0 : i] + ch * 8);
  };
  row = look(0);
  bf16x8 qf[C::DS];
  {
    const bf16_t* qp = a.q + (size_t)(s.q0 + tok) * a.ldq + (size_t)(kvh * G + rc % G) * HD + 8 * h;
#pragma unroll
    for (int ds = 0; ds < C::DS; ++ds) qf[ds] = *reinterpret_cast<const bf16x8*>(qp + ds * 16);
  }
  if (nt > 0) {
    aim(row);
#pragma unroll
    for (int i = 0; i < 2 * NQ; ++i) piece(0, i);
    next = look(1);
  }
  f32x16 o[C::DB];
#pragma unroll
  for (int d = 0; d < C::DB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
  for (int ds = 0; ds < C::DS; ++ds) asm volatile("" ::"v"(qf[ds]));

  for (int t = 0; t < nt; ++t) {
    const int k0 = ks + t * KV;
    unsigned long long ok;                          // keys of the tile that exist; the same in every wave
    if (ONE_PAGE) ok = __builtin_amdgcn_readfirstlane(row) < 0 ? 0ull : ke - k0 >= 64 ? ~0ull : (1ull << (ke - k0)) - 1;
    else ok = __ballot(row >= 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();                                // tile t is here, tile t - 1 is consumed: its stage takes t + 1
    unsigned char* kl = smem + (t & 1) * STAGE;
    unsigned char* vl = kl + TB;
    row = next;
    const bool more = t + 1 < nt;
    if (more) {
      aim(row);
      next = look(t + 2);
    }
    const bool edge = k0 + KV > clear || ok != ~0ull;        // uniform over the workgroup: some row may not see some key
    unsigned long long odd = 0;
    if (__builtin_expect(edge, 0)) {
      // V rows that do not exist become zeros (their p is 0, and 0 x NaN is not); rows with infinities or NaN are noted
      if (tid < 2) bad[tid] = 0;
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < NQ; ++i) {
        const int sidx = tid + 256 * i, trow = sidx / CPR;
        u32x4* x = reinterpret_cast<u32x4*>(vl + sidx * 16);
        const u32x4 y = *x;
        if (!((ok >> trow) & 1)) *x = u32x4{0u, 0u, 0u, 0u};
        else if (not_finite(y[0]) || not_finite(y[1]) || not_finite(y[2]) || not_finite(y[3])) atomicOr(&bad[trow >> 5], 1u << (trow & 31));
      }
      __syncthreads();
      odd = ((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)bad[1]) << 32) |
            (unsigned)__builtin_amdgcn_readfirstlane((int)bad[0]);
    }
    f32x16 st[2];
    float use = 0.f;
    const bool wanted = k0 < last_wave;
    if (!wanted && more) {
#pragma unroll
      for (int i = 0; i < 2 * NQ; ++i) piece(t + 1, i);
    }
    if (wanted) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) st[x][e] = 0.f;
      // fragments of the next k-step are requested ahead of a step's matrix instructions and its piece of DMA (2 NQ = DS)
      static_assert(2 * NQ == C::DS, "a piece a k-step");
      // (a wave's matrix phases go ahead of the co-resident workgroups' vector work: 1106 -> 1061 us on 2048 tokens over
      // 32 768 keys, 1142 -> 1129 on another card)
      __builtin_amdgcn_s_setprio(1);
      bf16x8 kf[2][2];
#pragma unroll
      for (int x = 0; x < 2; ++x) kf[0][x] = row_frag_sw<HD>(kl, x * 32, 0, lane);
#pragma unroll
      for (int ds = 0; ds < C::DS; ++ds) {
        if (ds + 1 < C::DS) {
#pragma unroll
          for (int x = 0; x < 2; ++x) kf[(ds + 1) & 1][x] = row_frag_sw<HD>(kl, x * 32, ds + 1, lane);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) st[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ds & 1][x], qf[ds], st[x], 0, 0, 0);
        if (more) piece(t + 1, ds);
      }
      if (__builtin_expect(edge, 0)) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const unsigned vis = seen_bits(a, s, tok, k0 + 32 * x) & (unsigned)(ok >> (32 * x));
#pragma unroll
          for (int e = 0; e < 16; ++e) st[x][e] = (vis >> acc_row(e, h)) & 1 ? st[x][e] : -INFINITY;
        }
      }
      __builtin_amdgcn_s_setprio(0);
      float mx = fmaxf(st[0][0], st[1][0]);
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, fmaxf(st[0][e], st[1][e]));
      mx = max_over32(mx) * sc;
      if (__any(mx > m_run + kSlack)) {
        const float mn = fmaxf(m_run, mx), f = fast_exp2(m_run - (mn == -INFINITY ? 0.f : mn));
        l_run *= f;
        m_run = mn;
#pragma unroll
        for (int d = 0; d < C::DB; ++d) o[d] = o[d] * f;
      }
      use = m_run == -INFINITY ? 0.f : m_run;
    }
    if (__builtin_expect(odd != 0, 0)) {
      // keys with infinities or NaN in V: added on their own to the rows that see them, then zeros for the product below
      if (wanted) {
#pragma unroll 1
        for (unsigned long long left = odd; left; left &= left - 1) {
          const int kk = __ffsll(left) - 1;
          float x = 0.f;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (e == (kk >> 5) * 16 + (kk & 3) + 4 * ((kk & 31) >> 3)) x = st[e >> 4][e & 15];
          x = fast_exp2(__builtin_fmaf(__shfl(x, ((kk >> 2) & 1) * 32 + (lane & 31), 64), sc, -use));
          if (x != 0.f) {
#pragma unroll
            for (int d = 0; d < C::DB; ++d)
#pragma unroll
              for (int r4 = 0; r4 < 4; ++r4) {
                const u32x2 y = *reinterpret_cast<const u32x2*>(vl + kk * RB + (((d * 4 + r4) ^ swz_key<HD>(kk)) << 4) + 8 * h);
                o[d][4 * r4] += x * lo_bf(y[0]); o[d][4 * r4 + 1] += x * hi_bf(y[0]);
                o[d][4 * r4 + 2] += x * lo_bf(y[1]); o[d][4 * r4 + 3] += x * hi_bf(y[1]);
              }
          }
        }
      }
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < NQ; ++i)
        if ((odd >> ((tid + 256 * i) / CPR)) & 1) *reinterpret_cast<u32x4*>(vl + (tid + 256 * i) * 16) = u32x4{0u, 0u, 0u, 0u};
      __syncthreads();
    }
    if (wanted) {
      // 16 keys at a time: their exponentials, then the matrix instructions that take them
      __builtin_amdgcn_s_setprio(1);
      const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
      float rs = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          bf16x8 pf;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            pf[e] = (__bf16)fast_exp2(__builtin_fmaf(st[x][8 * z + e], sc, -use));
          }
          // the row's sum takes the probabilities as the product does, rounded to bf16 (one rounding, to nearest, so that
          // neither side leans); two to an instruction, in fp32 (adding the unrounded ones: 1136 -> 1108 us on 2048 tokens
          // over 32 768 keys)
#pragma unroll
          for (int e = 0; e < 8; e += 2) rs = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{pf[e], pf[e + 1]}, one, rs, false);
#pragma unroll
          for (int d = 0; d < C::DB; ++d)
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_frag_sw<HD>(vl, x * 32, z, d, lane), pf, o[d], 0, 0, 0);
        }
      l_run += rs;
      __builtin_amdgcn_s_setprio(0);
    }
  }
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  if (r >= rows) return;
  const int tq = s.q0 + tok, head = kvh * G + rc % G;
  if (alone) {
    const float inv = l_tot > 0.f ? 1.0f / l_tot : (l_tot == 0.f ? 0.f : l_tot);
    bf16_t* op = a.out + (size_t)tq * a.ldo + (size_t)head * HD;
#pragma unroll
    for (int d = 0; d < C::DB; ++d)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        u32x2 y;
        y[0] = pack2bf(o[d][4 * r4] * inv, o[d][4 * r4 + 1] * inv);
        y[1] = pack2bf(o[d][4 * r4 + 2] * inv, o[d][4 * r4 + 3] * inv);
        *reinterpret_cast<u32x2*>(op + d * 32 + 8 * r4 + 4 * h) = y;
      }
  } else {
    const size_t part = (size_t)blockIdx.x * 128 + (r - t0);
#pragma unroll
    for (int d = 0; d < C::DB; ++d)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        *reinterpret_cast<f32x4*>(a.part_o + part * HD + d * 32 + 8 * r4 + 4 * h) =
            f32x4{o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]};
    if (h == 0) { a.part_ml[part * 2] = m_run; a.part_ml[part * 2 + 1] = l_tot; }
  }
}

// out = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over the shares of a row's sequence, in a fixed order: one workgroup
// per (token, head, slice of 32 columns); 8 threads read a share's columns, the others every following share, and the
// groups' sums are added in order.  Slices: 512 shares of 8 rows 20.4 us a call, 24.5 with a workgroup a row; 32 of 512 rows
// 208.4 against 206.8.
constexpr int kMergeThreads = 256;
template <int HD>
__global__ __launch_bounds__(kMergeThreads) void attn_paged_merge_kernel(PagedArgs a) {
  constexpr int COLS = 32, TPG = COLS / 4, NG = kMergeThreads / TPG, NSL = HD / COLS;
  __shared__ float wgt[1024];
  __shared__ __attribute__((aligned(16))) float acc[NG][COLS];
  __shared__ float red[4], sum[4];
  const int id = blockIdx.x / NSL, t = id / a.Hq, h = id % a.Hq, col0 = blockIdx.x % NSL * COLS, tid = threadIdx.x;
  const Seq s(a, seq_of(a, t));
  if (t < s.q0 || t >= s.q0 + min(s.n, a.max_q)) return;
  const int parts = min(a.splits, (s.len + a.split_keys - 1) / a.split_keys);
  if (parts <= 1) return;                           // written by its only share
  const float* ml = a.part_ml + (size_t)id * a.splits * 2;
  const float* po = a.part_o + (size_t)id * a.splits * HD + col0;
  float M = -INFINITY;
  for (int i = tid; i < parts; i += kMergeThreads) M = fmaxf(M, ml[2 * i]);
  M = wave_max(M);
  if ((tid & 63) == 0) red[tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const int g = tid / TPG, c = (tid % TPG) * 4;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  float L = 0.f;
  for (int i0 = 0; i0 < parts; i0 += 1024) {
    const int np = min(1024, parts - i0);
    __syncthreads();
    for (int i = tid; i < np; i += kMergeThreads) {
      const float f = M == -INFINITY ? 0.f : fast_exp2(ml[2 * (i0 + i)] - M);
      wgt[i] = f;
      L += ml[2 * (i0 + i) + 1] * f;
    }
    __syncthreads();
#pragma unroll 4
    for (int i = g; i < np; i += NG) {              // (a share that saw nothing of this row has weight 0 and zeros)
      const f32x4 x = *reinterpret_cast<const f32x4*>(po + (size_t)(i0 + i) * HD + c);
      y += x * wgt[i];
    }
  }
  *reinterpret_cast<f32x4*>(&acc[g][c]) = y;
  L = wave_sum(L);
  if ((tid & 63) == 0) sum[tid >> 6] = L;
  __syncthreads();
  if (tid >= COLS) return;
  L = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < NG; ++i) v += acc[i][tid];
  const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);
  a.out[(size_t)t * a.ldo + (size_t)h * HD + col0 + tid] = f2bf(v * inv);
}

// y += sum_j f[lane j] * x[j * step ..] over up to 64 shares, eight loads in flight: the first eight go out with `load`, before
// the weights f are there
template <int CPL>
struct ShareSum {
  typedef __attribute__((ext_vector_type(CPL))) float fv;
  fv v[8];
  __device__ __forceinline__ void load(const float* x, size_t step, int parts, int j = 0) {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const fv*>(x + (size_t)min(j + u, parts - 1) * step);
  }
  __device__ __forceinline__ void add(float (&y)[CPL], const float* x, size_t step, int parts, float f) {
    for (int j = 0; j < parts; j += 8) {
      if (j) load(x, step, parts, j);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(f), j + u));
        if (j + u < parts) {                        // (not by w = 0 alone: the repeated last share may be infinite)
#pragma unroll
          for (int c = 0; c < CPL; ++c) y[c] += v[u][c] * w;
        }
      }
    }
  }
};

// the same for few shares: a wave a row, HD / 64 columns a lane, four rows a workgroup
template <int HD>
__global__ __launch_bounds__(256) void attn_paged_merge_few_kernel(PagedArgs a) {
  constexpr int CPL = HD / 64;
  const int lane = threadIdx.x & 63;
  const int id = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  if (id >= a.T * a.Hq) return;
  const int t = id / a.Hq, h = id % a.Hq;
  const Seq s(a, seq_of(a, t));
  if (t < s.q0 || t >= s.q0 + min(s.n, a.max_q)) return;
  const int parts = min(a.splits, (s.len + a.split_keys - 1) / a.split_keys);
  if (parts <= 1) return;
  const float* ml = a.part_ml + (size_t)id * a.splits * 2;
  const float* po = a.part_o + (size_t)id * a.splits * HD + lane * CPL;
  float m = lane < parts ? ml[2 * lane] : -INFINITY, l = lane < parts ? ml[2 * lane + 1] : 0.f;
  ShareSum<CPL> sum;
  sum.load(po, HD, parts);
  const float M = wave_max(m);
  const float f = M == -INFINITY ? 0.f : fast_exp2(m - M);
  const float L = wave_sum(l * f);
  const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);
  float y[CPL];
#pragma unroll
  for (int c = 0; c < CPL; ++c) y[c] = 0.f;
  sum.add(y, po, HD, parts, f);
  bf16_t* op = a.out + (size_t)t * a.ldo + (size_t)h * HD + lane * CPL;
  if (CPL == 2) *reinterpret_cast<unsigned*>(op) = pack2bf(y[0] * inv, y[CPL - 1] * inv);
  else *op = f2bf(y[0] * inv);
}

// the same for the tile kernel's shares: a workgroup is a token and 4 NH heads, a wave NH of them, so that what leads to the
// shares (four loads that wait for each other) is gone through once and the heads' loads are in flight together
template <int HD, int NH>
__global__ __launch_bounds__(256) void attn_paged_merge_tiles_kernel(PagedArgs a) {
  constexpr int CPL = HD / 64;
  const int q = a.shares[0], hb = (a.Hq + 4 * NH - 1) / (4 * NH), t = (int)blockIdx.x / hb, b = seq_of(a, t);
  if (!q) return;                                   // no sequence was shared out
  const int lane = threadIdx.x & 63, G = a.Hq / a.Hkv;
  const int h0 = ((int)blockIdx.x % hb) * 4 * NH + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) * NH;
  const Seq s(a, b);
  const int i = t - s.q0, parts = (((s.len + 63) >> 6) + q - 1) / q, first = a.shares[1 + b];
  if (i < 0 || i >= min(s.n, a.max_q) || parts <= 1) return;
  const size_t step = (size_t)a.Hkv * 128;
  size_t p0[NH];
  float m[NH], l[NH];
#pragma unroll
  for (int x = 0; x < NH; ++x) {
    const int h = min(h0 + x, a.Hq - 1), r = i * G + h % G;
    p0[x] = (size_t)(first + (r >> 7) * parts * a.Hkv + h / G) * 128 + (r & 127);
    const float* ml = a.part_ml + 2 * (p0[x] + min(lane, parts - 1) * step);
    m[x] = ml[0];
    l[x] = ml[1];
  }
  ShareSum<CPL> sum[NH];
#pragma unroll
  for (int x = 0; x < NH; ++x) sum[x].load(a.part_o + p0[x] * HD + lane * CPL, step * HD, parts);
#pragma unroll
  for (int x = 0; x < NH; ++x) {
    const float M = wave_max(m[x]);
    const float f = M == -INFINITY || lane >= parts ? 0.f : fast_exp2(m[x] - M);
    const float L = wave_sum(lane < parts ? l[x] * f : 0.f);
    const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);
    float y[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) y[c] = 0.f;
    sum[x].add(y, a.part_o + p0[x] * HD + lane * CPL, step * HD, parts, f);
    if (h0 + x < a.Hq) {
      bf16_t* op = a.out + (size_t)t * a.ldo + (size_t)(h0 + x) * HD + lane * CPL;
      if (CPL == 2) *reinterpret_cast<unsigned*>(op) = pack2bf(y[0] * inv, y[CPL - 1] * inv);
      else *op = f2bf(y[0] * inv);
    }
  }
}

// shape of a launch: host arithmetic on the sizes alone
struct Plan {
  int mt, waves, splits, split_keys, merge_heads;   // mt: 16-row groups of the stream kernel, 8 = the tile kernel
  int64_t grid, merge, header, parts, ws;           // workgroups of both launches; floats of the header, parts, floats altogether
};
inline Plan plan_of(int64_t B, int64_t T, int64_t max_q, int64_t max_ctx, int64_t Hq, int64_t Hkv, int64_t hd) {
  Plan p{};
  const int64_t rows = (max_q < T ? max_q : T) * (Hq / Hkv);       // (no sequence has more new tokens than there are)
  // 20 rows of width 128 over 2 x 8192 (16 x 1024) keys: 23.2 (18.2) us by two 16-row groups, 24.7 (20.7) by tiles; over
  // 8 x 4096: 39.0, 36.6.  24 rows of width 64 over 8 x 4096: 41.5 by two groups, 39.0 by tiles.  4 rows: 18 against 24.
  p.mt = rows <= 16 ? 1 : rows <= 32 && hd == 128 ? 2 : 8;
  if (p.mt == 8) {
    const int64_t groups = B * Hkv * ((rows + 127) / 128);
    // shares are cut on the device; no sequence of up to four 64-key tiles is, nor any where there is work for two rounds
    const int64_t slots = hd == 64 ? kTileSlots<64> : kTileSlots<128>;
    const bool shared = max_ctx > 256 && T * Hq < 128 * 2 * slots;
    p.splits = shared ? 2 : 1;
    p.grid = shared && groups < 2 * slots ? 2 * slots : groups;
    p.header = shared ? (B + 64) / 64 * 64 : 0;
    p.parts = shared ? 2 * slots * 128 : 0;
    // a wave a row while every row's wave is resident at once (256 CUs x 32): 160 rows x 8 heads of 50 shares 33.2 -> 31.4 us
    // a call, 89 x 2 x 8 31.3 -> 28.6; beyond, two rows a wave: 1000 x 16 48.6, 51.3 by one
    p.merge_heads = T * Hq <= 8192 ? 1 : 2;
    p.merge = shared ? T * ((Hq + 4 * p.merge_heads - 1) / (4 * p.merge_heads)) : 0;
  } else {
    // shares of the keys: as many as fill the 512 workgroups that the CUs hold at two each, none under 128 keys (a piece
    // for each wave) and none over 512: the lengths of a batch differ, and small shares even that out (48 sequences of
    // 700 to 8192: 150 us with 1024 keys, 140 with 512)
    const int64_t groups = B * Hkv;
    int64_t keys = (max_ctx * groups + 511) / 512;
    keys = (keys + 127) / 128 * 128;
    keys = keys < 128 ? 128 : keys > 512 ? 512 : keys;
    p.waves = 4;
    // No shares and no merge, but eight waves, where that costs less than a merge (3 us): what the CUs without a workgroup
    // would have taken off the longest sequence's K and V, at the 46 GB/s that a CU reads, is 140 KB; and not above 512 KB,
    // as lengths differ.  (32 over 8 of 128: 24 x 512 keys 12.7 us, 16.0 by shares; 24 x 1024 21.0, 25.4; 64 x 771 35.9,
    // 39.7; 8 x 256 6.8, 7.8; but 8 x 512 9.6, 7.8.  16 of 64: 8 x 512 6.6, 8.2; 1 x 512 6.1, 7.0; 1 x 771 8.2, 7.2)
    const int64_t bytes = max_ctx * hd * 4, idle = groups < 256 ? 256 - groups : 0;
    if (p.mt == 1 && keys < max_ctx && bytes <= (512 << 10) && bytes * idle <= 256 * (140 << 10)) {
      keys = max_ctx;
      p.waves = 8;
    }
    p.split_keys = (int)keys;
    p.splits = (int)((max_ctx + keys - 1) / keys);
    p.grid = groups * p.splits;
    p.parts = p.splits > 1 ? T * Hq * p.splits : 0;
    // few shares: a wave a row (7 shares of 32 rows 8.2 us a call, 8.8 by workgroups; 4 of 1536 rows 83.7, 90.9; but 64 of
    // 32 rows 21.1, 18.4, and 32 of 128 rows 48.2, 47.0)
    p.merge = p.splits == 1 ? 0 : p.splits <= 16 ? (T * Hq + 3) / 4 : T * Hq * (hd / 32);
  }
  p.ws = p.header + p.parts * (hd + 2);
  return p;
}

inline bool odd16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace

extern "C" int zk_kv_append_paged(const void* qkv, const float* cos_t, const float* sin_t, void* q_out, void* k_cache,
                                  void* v_cache, const int32_t* positions, const int32_t* slots, int64_t T, int64_t Hq,
                                  int64_t Hkv, int64_t head_dim, int64_t rot_dim, int64_t table_rows, int64_t ldqkv,
                                  int64_t ldq, int64_t cache_rows, int interleaved, hipStream_t stream) {
  if (T < 0 || T > 0x7FFFFFFF || Hq <= 0 || Hkv <= 0 || Hq % Hkv || (head_dim != 64 && head_dim != 128)) return ZK_EINVAL;
  if (zk_too_many(T, 256)) return ZK_EINVAL;
  if ((Hq + 2 * Hkv) * head_dim > (1 << 24)) return ZK_EINVAL;
  if (rot_dim < 16 || (rot_dim & 15) || rot_dim > head_dim || table_rows <= 0 || table_rows > 0x7FFFFFFF) return ZK_EINVAL;
  if (cache_rows <= 0 || cache_rows > 0x7FFFFFFF || (ldqkv & 7) || (ldq & 7)) return ZK_EINVAL;
  if (ldqkv < (Hq + 2 * Hkv) * head_dim || ldq < Hq * head_dim) return ZK_EINVAL;
  if (!qkv || !cos_t || !sin_t || !q_out || !k_cache || !v_cache || !positions || !slots) return ZK_EINVAL;
  if (odd16(qkv) || odd16(cos_t) || odd16(sin_t) || odd16(q_out) || odd16(k_cache) || odd16(v_cache)) return ZK_EINVAL;
  if (T == 0) return ZK_OK;
  auto kern = head_dim == 128 ? kv_append_paged_kernel<128> : kv_append_paged_kernel<64>;
  hipLaunchKernelGGL(kern, dim3((unsigned)T), dim3(256), 0, stream, (const bf16_t*)qkv, cos_t, sin_t, (bf16_t*)q_out,
                     (bf16_t*)k_cache, (bf16_t*)v_cache, positions, slots, (int)Hq, (int)Hkv, (int)rot_dim,
                     (int)table_rows, (long long)ldqkv, (long long)ldq, (long long)cache_rows, interleaved ? 1 : 0);
  ZK_CHECK_LAUNCH();
  return ZK_OK;
}

extern "C" int zk_attn_paged_ws(int64_t B, int64_t T, int64_t max_q, int64_t max_ctx, int64_t Hq, int64_t Hkv,
                                int64_t head_dim, int64_t* ws_floats) {
  if (!ws_floats || B <= 0 || T < 0 || max_q <= 0 || max_ctx <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return ZK_EINVAL;
  if ((head_dim != 64 && head_dim != 128) || T >= kMaxRows || max_q > 0x7FFFFFFF || max_ctx > 0x7FFFFF00) return ZK_EINVAL;
  if (B >= kMaxRows || Hq > (1 << 17) || B * Hkv > (1 << 28) || T * Hq > 0x7FFFFFFF) return ZK_EINVAL;
  const Plan p = T ? plan_of(B, T, max_q, max_ctx, Hq, Hkv, head_dim) : Plan{};
  if (zk_too_many(p.grid, p.waves == 8 ? 512 : 256) || zk_too_many(p.merge, kMergeThreads)) return ZK_EINVAL;
  *ws_floats = p.ws;
  return ZK_OK;
}

extern "C" int zk_attn_paged(const void* q, const void* k_cache, const void* v_cache, void* out, const int32_t* page_table,
                             const int32_t* ctx_lens, const int32_t* cu_q, const int64_t* tree_mask, float* ws,
                             int64_t ws_floats, int64_t T, int64_t B, int64_t max_q, int64_t max_ctx, int64_t Hq,
                             int64_t Hkv, int64_t head_dim, int64_t page_size, int64_t n_pages, int64_t table_cols,
                             int64_t ld_table, int64_t mask_words, int64_t ldq, int64_t ldo, float scale,
                             hipStream_t stream) {
  int64_t need = 0;
  const int rc = zk_attn_paged_ws(B, T, max_q, max_ctx, Hq, Hkv, head_dim, &need);
  if (rc != ZK_OK) return rc;
  if (page_size <= 0 || n_pages <= 0 || table_cols <= 0 || ld_table < table_cols) return ZK_EINVAL;
  if (page_size > 0x7FFFFFFF || n_pages > 0x7FFFFFFF || ld_table > 0x7FFFFFFF) return ZK_EINVAL;
  if (n_pages * page_size > 0x7FFFFFFF || !(scale > 0.f && scale < INFINITY)) return ZK_EINVAL;
  if ((ldq & 7) || (ldo & 7) || ldq < Hq * head_dim || ldo < Hq * head_dim) return ZK_EINVAL;
  if (!q || !k_cache || !v_cache || !out || !page_table || !ctx_lens || !cu_q) return ZK_EINVAL;
  if (tree_mask && (mask_words <= 0 || mask_words > (1 << 20))) return ZK_EINVAL;
  if (odd16(q) || odd16(k_cache) || odd16(v_cache) || odd16(out) || (need > 0 && (!ws || odd16(ws) || ws_floats < need)))
    return ZK_EINVAL;
  if (T == 0) return ZK_OK;
  const Plan p = plan_of(B, T, max_q, max_ctx, Hq, Hkv, head_dim);
  int lg = 0;                                       // page_mul: the 31-bit reciprocal, rounded up (exact below 2^31)
  while ((int64_t)1 << lg < page_size) ++lg;
  const unsigned mul = (unsigned)((((unsigned long long)1 << (31 + lg)) / (unsigned long long)page_size) + 1);
  float* part_o = p.splits > 1 ? ws + p.header : nullptr;
  PagedArgs a{(const bf16_t*)q, (const bf16_t*)k_cache, (const bf16_t*)v_cache, (bf16_t*)out, page_table, ctx_lens, cu_q,
              (const unsigned long long*)tree_mask, part_o, part_o ? part_o + p.parts * head_dim : nullptr, (int*)ws, (int)T,
              (int)B, (int)max_q, (int)Hq, (int)Hkv, (int)page_size, (int)n_pages, (int)table_cols, (int)ld_table,
              (int)mask_words, p.splits, p.split_keys, mul, (unsigned)(31 + lg),
              (long long)ldq, (long long)ldo, scale};
  const bool one_page = page_size % 64 == 0;
  void (*kern)(PagedArgs) =
      head_dim == 128 ? (p.mt == 1 ? (p.waves == 4 ? attn_paged_stream_kernel<128, 1, 4> : attn_paged_stream_kernel<128, 1, 8>) : p.mt == 2 ? attn_paged_stream_kernel<128, 2, 4> : one_page ? attn_paged_tile_kernel<128, true> : attn_paged_tile_kernel<128, false>)
                      : (p.mt == 1 ? (p.waves == 4 ? attn_paged_stream_kernel<64, 1, 4> : attn_paged_stream_kernel<64, 1, 8>) : one_page ? attn_paged_tile_kernel<64, true> : attn_paged_tile_kernel<64, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)p.grid), dim3(p.waves == 8 ? 512 : 256), 0, stream, a);
  if (p.splits > 1) {
    const bool one = p.merge_heads == 1, few = p.splits <= 16;
    void (*merge)(PagedArgs) =
        p.mt == 8 ? (head_dim == 128 ? (one ? attn_paged_merge_tiles_kernel<128, 1> : attn_paged_merge_tiles_kernel<128, 2>)
                                     : (one ? attn_paged_merge_tiles_kernel<64, 1> : attn_paged_merge_tiles_kernel<64, 2>))
                  : (head_dim == 128 ? (few ? attn_paged_merge_few_kernel<128> : attn_paged_merge_kernel<128>)
                                     : (few ? attn_paged_merge_few_kernel<64> : attn_paged_merge_kernel<64>));
    hipLaunchKernelGGL(merge, dim3((unsigned)p.merge), dim3(kMergeThreads), 0, stream, a);
  }
  ZK_CHECK_LAUNCH();
  return ZK_OK;
}
