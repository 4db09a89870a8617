// Serving operators over a paged key / value cache: append with rotation, attention of new tokens.
//
// The cache of one layer is two bf16 arrays [n_pages][page_size][Hkv * hd] (keys after rotation, values); a sequence
// owns the pages its row of the page table names, so its cached row r is row r % page_size of page table[r / page_size].
// The layout is the token-major one of the contiguous caches (zk_attn_decode): the new rows of a token are one store,
// and a contiguous cache [B][rows][Hkv * hd] is the special case of one page per sequence.
// Every index that comes from device memory (slots, positions, page numbers, lengths) is checked in the kernel against
// the sizes the host passed: nothing is read or written outside the arrays whatever the tables hold.
#include "common.h"
#include "../../include/zero_hip.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// =========================================================================================
// append: one workgroup per token, a unit of work is 16 values of a head (two 16-byte chunks) that turn by 8 angles.
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
  int T, B, Hq, Hkv, page_size, n_pages, table_cols, ld_table, mask_words;
  long long ldq, ldo;
  float scale;
};

// =========================================================================================
// attention, one wave per (new token, query head): 64 keys at a time, a lane scores one key, then owns hd / 64 output
// columns.  Running maximum and sum of the softmax in fp32.
// =========================================================================================
template <int HD>
__global__ __launch_bounds__(64) void attn_paged_rows_kernel(PagedArgs a) {
  constexpr int CPL = HD / 64;
  __shared__ float qs[HD];
  __shared__ float ps[64];
  __shared__ long long rows[64];
  const int lane = threadIdx.x, t = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, kvh = h / (a.Hq / a.Hkv);
  int lo = 0, hi = a.B;                             // last sequence that starts at or before row t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= t) lo = mid; else hi = mid;
  }
  const int b = lo, q0 = a.cu[b], q1 = a.cu[b + 1];
  if (t < q0 || t >= q1) return;                    // rows behind the last sequence stay as they are
  const int len = min(max(a.ctx[b], 0), (int)min((long long)a.table_cols * a.page_size, 0x7FFFFFFFLL));
  const long long first = (long long)a.ctx[b] - (q1 - q0);
  const int kvw = a.Hkv * HD, i = t - q0;
  for (int d = lane; d < HD; d += 64) qs[d] = bf2f(a.q[(size_t)t * a.ldq + h * HD + d]) * (a.scale * kLog2e);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[CPL];
#pragma unroll
  for (int c = 0; c < CPL; ++c) acc[c] = 0.f;
  for (int k0 = 0; k0 < len; k0 += 64) {
    const int key = k0 + lane;
    bool seen = key < len;
    const long long j = (long long)key - first;     // which new token this row is (negative: a row before them)
    if (seen && j >= 0) {
      if (a.mask) seen = (j >> 6) < a.mask_words && ((a.mask[(size_t)t * a.mask_words + (j >> 6)] >> (j & 63)) & 1);
      else seen = j <= i;
    }
    long long r = -1;
    if (seen) {
      const int pg = a.table[(size_t)b * a.ld_table + key / a.page_size];
      if (pg >= 0 && pg < a.n_pages) r = (long long)pg * a.page_size + key % a.page_size;
    }
    float s = -INFINITY;
    if (r >= 0) {
      const bf16_t* kp = a.k + (size_t)r * kvw + kvh * HD;
      s = 0.f;
      for (int c = 0; c < HD / 8; ++c) {
        const u32x4 kr = *reinterpret_cast<const u32x4*>(kp + c * 8);
#pragma unroll
        for (int e = 0; e < 4; ++e) s += lo_bf(kr[e]) * qs[c * 8 + 2 * e] + hi_bf(kr[e]) * qs[c * 8 + 2 * e + 1];
      }
    }
    const float mn = fmaxf(m, wave_max(s));
    const float base = mn == -INFINITY ? 0.f : mn;
    const float p = r >= 0 ? __builtin_amdgcn_exp2f(s - base) : 0.f;
    const float f = __builtin_amdgcn_exp2f(m - base);
    __syncthreads();
    ps[lane] = p;
    rows[lane] = r;
    __syncthreads();
    l = l * f + wave_sum(p);
    m = mn;
#pragma unroll
    for (int c = 0; c < CPL; ++c) acc[c] *= f;
    for (int kk = 0; kk < 64; ++kk) {
      const long long rr = rows[kk];
      if (rr < 0) continue;
      const bf16_t* vp = a.v + (size_t)rr * kvw + kvh * HD + lane * CPL;
#pragma unroll
      for (int c = 0; c < CPL; ++c) acc[c] += ps[kk] * bf2f(vp[c]);
    }
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;       // a row that sees nothing is zero
#pragma unroll
  for (int c = 0; c < CPL; ++c) a.out[(size_t)t * a.ldo + h * HD + lane * CPL + c] = f2bf(acc[c] * inv);
}

inline bool odd16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace

extern "C" int zk_kv_append_paged(const void* qkv, const float* cos_t, const float* sin_t, void* q_out, void* k_cache,
                                  void* v_cache, const int32_t* positions, const int32_t* slots, int64_t T, int64_t Hq,
                                  int64_t Hkv, int64_t head_dim, int64_t rot_dim, int64_t table_rows, int64_t ldqkv,
                                  int64_t ldq, int64_t cache_rows, int interleaved, hipStream_t stream) {
  if (T < 0 || T > 0x7FFFFFFF || Hq <= 0 || Hkv <= 0 || Hq % Hkv || (head_dim != 64 && head_dim != 128)) return ZK_EINVAL;
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
  if (head_dim != 64 && head_dim != 128) return ZK_EINVAL;
  *ws_floats = 0;
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
  if (T > 0x7FFFFFFF || B > 0x7FFFFFFE || page_size > 0x7FFFFFFF || n_pages > 0x7FFFFFFF || ld_table > 0x7FFFFFFF) return ZK_EINVAL;
  if (n_pages * page_size > 0x7FFFFFFF || T * Hq > 0x7FFFFFFF || Hkv * head_dim > (1 << 24)) return ZK_EINVAL;
  if ((ldq & 7) || (ldo & 7) || ldq < Hq * head_dim || ldo < Hq * head_dim) return ZK_EINVAL;
  if (!q || !k_cache || !v_cache || !out || !page_table || !ctx_lens || !cu_q) return ZK_EINVAL;
  if (tree_mask && (mask_words <= 0 || mask_words > (1 << 20))) return ZK_EINVAL;
  if (odd16(q) || odd16(k_cache) || odd16(v_cache) || odd16(out) || (need > 0 && (!ws || odd16(ws) || ws_floats < need)))
    return ZK_EINVAL;
  if (T == 0) return ZK_OK;
  PagedArgs a{(const bf16_t*)q, (const bf16_t*)k_cache, (const bf16_t*)v_cache, (bf16_t*)out, page_table, ctx_lens, cu_q,
              (const unsigned long long*)tree_mask, (int)T, (int)B, (int)Hq, (int)Hkv, (int)page_size, (int)n_pages,
              (int)table_cols, (int)ld_table, (int)mask_words, (long long)ldq, (long long)ldo, scale};
  auto kern = head_dim == 128 ? attn_paged_rows_kernel<128> : attn_paged_rows_kernel<64>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(T * Hq)), dim3(64), 0, stream, a);
  ZK_CHECK_LAUNCH();
  return ZK_OK;
}
