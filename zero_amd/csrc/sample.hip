// Drawing the next token of every row of bf16 logits: temperature, top-k, top-p, min-p, from a given number u.
//
// Definition (per row).  Tokens in falling order of their logit, equal logits by the lower index; w_r = e^((l_r - max) / T).
//   top-k keeps the first k; top-p the shortest prefix whose sum reaches p times the sum of what top-k kept; min-p the
//   tokens with w >= min_p.  All three are prefixes of one order, so the kept set is the shortest of them, and the token
//   drawn is the first whose running sum exceeds u * Z, Z = the kept sum.  logprob = log(w / Z).
//
// bf16 logits have at most 65 281 different values that can be drawn, so the sorted row is its HISTOGRAM: bin d (0 = the
// largest value's bin) holds how many tokens have that value, a bin of c tokens adds c * w(d) to the running sum, and no
// sort of 10^5 tokens is needed.  One workgroup owns a row; its bins live in LDS as 32-bit counts.  Sums are formed in
// 64 bits over the occupied bins only (a few thousand exponentials instead of one per token), so that the token does not
// depend on how a sum was split: the running sum of 10^5 weights in 32 bits would move its borders by more than the
// weight of a rare token.
//
// 39 936 bins (156 KiB of the CU's 160) instead of 65 281: a token further below the maximum than the last bin differs
// from it by more than 2^28 (two bf16 of one sign are at most 32 640 values apart, so the signs differ and one of the
// two magnitudes is beyond 2^28), and its weight is zero at every temperature up to 2^20, the largest one used.
#include "common.h"
#include "../../include/zero_hip.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBpt = 39, kBins = kThreads * kBpt;   // bins per thread: odd, so that thread-contiguous bins are read without bank conflicts
constexpr int kChunks = 16;                         // 16-byte chunks of the row a thread holds in registers
constexpr int kRound = kThreads * 8 * kChunks;      // tokens of one register-held part of a row
constexpr float kMaxTemperature = 1048576.0f;

struct SampleArgs {
  const bf16_t* logits;
  const float *u, *temperature_rows, *top_p_rows, *min_p_rows;
  const int* top_k_rows;
  float temperature, top_p, min_p;
  int top_k;
  long long* tokens;
  float* logprobs;
  long long V, ld;
  int vec;                                          // rows are 16-byte aligned
};

// place of a logit in falling order (0 = largest): -0 is +0.  0x7F = +inf, 0xFF80 = -inf; beyond these: NaN
__device__ __forceinline__ int falling(unsigned b) {
  const unsigned m = b & 0x7FFFu;
  return (b & 0x8000u) && m ? (int)(0x7FFFu + m) : (int)(0x7FFFu - m);
}
constexpr int kTop = 0x7F, kBottom = 0x7FFF + 0x7F80;   // +inf, -inf
__device__ __forceinline__ double value_of(int d) {
  const unsigned b = d <= 0x7FFF ? (unsigned)(0x7FFF - d) : (0x8000u | (unsigned)(d - 0x7FFF));
  return (double)bf2f((bf16_t)b);
}

struct Row {
  u32x4 r[kChunks];
  // chunk c of the part: tokens part + (c * kThreads + tid) * 8 ..
  __device__ __forceinline__ void load(const SampleArgs& a, const bf16_t* row, long long part, int tid) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const long long i = part + (long long)(c * kThreads + tid) * 8;
      u32x4 x = {0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u};     // -inf past the row's end
      if (i + 8 <= a.V && a.vec) {
        x = *reinterpret_cast<const u32x4*>(row + i);
      } else if (i < a.V) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < a.V) {
            const unsigned v = row[i + e];
            x[e >> 1] = e & 1 ? (x[e >> 1] & 0xFFFFu) | (v << 16) : (x[e >> 1] & 0xFFFF0000u) | v;
          }
      }
      r[c] = x;
    }
  }
  __device__ __forceinline__ int place(int c, int e) const {
    return falling((r[c][e >> 1] >> ((e & 1) * 16)) & 0xFFFFu);
  }
};

__device__ __forceinline__ double shfl_up_d(double v, int o) {
  return __hiloint2double(__shfl_up(__double2hiint(v), o, 64), __shfl_up(__double2loint(v), o, 64));
}

// sum of v over the threads before this one; upto = with this one's (the same bits as the next thread's `before`, so that
// exactly one thread holds a border); total = over all.  Fixed order: equal inputs give equal bits.
template <class T, class Up>
__device__ __forceinline__ T block_before(T v, T* waves, T& upto, T& total, Up up) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T x = up(inc, o);
    if (lane >= o) inc += x;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = inc;
  __syncthreads();
  T base = 0;
  for (int w = 0; w < wave; ++w) base += waves[w];
  total = base;
  for (int w = wave; w < kWaves; ++w) total += waves[w];
  T ex = up(inc, 1);
  if (lane == 0) ex = 0;
  upto = base + inc;
  return base + ex;
}

__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned hist[kBins];
  __shared__ double wsum[kWaves], shared_mass;
  __shared__ unsigned wcnt[kWaves];
  __shared__ int wtop[kWaves], wnan[kWaves], pick_bin, pick_rank;
  __shared__ unsigned matches[kChunks * kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long b = blockIdx.x;
  const bf16_t* row = a.logits + b * a.ld;
  float Tf = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
  const int top_k = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
  const double top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
  const double min_p = a.min_p_rows ? a.min_p_rows[b] : a.min_p;
  const bool greedy = !(Tf > 0.f);
  Tf = fminf(Tf, kMaxTemperature);
  const double T = greedy ? 1.0 : (double)Tf;
  const unsigned long long limit = greedy ? 1ull : top_k > 0 ? (unsigned long long)top_k : ~0ull;

  Row x;
  const bool resident = a.V <= kRound;
  if (resident) x.load(a, row, 0, tid);
  for (int i = tid; i < kBins / 4; i += kThreads) reinterpret_cast<u32x4*>(hist)[i] = u32x4{0u, 0u, 0u, 0u};
  // the largest logit, and whether any is NaN
  int top = kBottom, nan = 0;
  for (long long part = 0; part < a.V; part += kRound) {
    if (!resident) x.load(a, row, part, tid);
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = x.place(c, e);
        nan |= d < kTop || d > kBottom;
        top = min(top, d);
      }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { top = min(top, __shfl_xor(top, o, 64)); nan |= __shfl_xor(nan, o, 64); }
  if (lane == 0) { wtop[wave] = top; wnan[wave] = nan; }
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) { top = min(top, wtop[w]); nan |= wnan[w]; }
  if (nan || top >= kBottom) {                      // a NaN, or no token that can be drawn
    if (tid == 0) {
      a.tokens[b] = -1;
      a.logprobs[b] = nan ? __builtin_nanf("") : -INFINITY;
    }
    return;
  }
  for (long long part = 0; part < a.V; part += kRound) {
    if (!resident) x.load(a, row, part, tid);
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = x.place(c, e);
        if (d < kBottom && d - top < kBins) atomicAdd(&hist[d - top], 1u);
      }
  }
  __syncthreads();
  // weight of bin i (a maximum of +inf has the only weight)
  const double vtop = value_of(top);
  auto weight = [&](int i) { return i == 0 ? 1.0 : exp((value_of(top + i) - vtop) / T); };
  const int i0 = tid * kBpt;
  unsigned cnt = 0;
  double mass = 0.0, mass_mp = 0.0;
  for (int i = i0; i < i0 + kBpt; ++i) {
    const unsigned c = hist[i];
    if (!c) continue;
    const double w = weight(i), cw = (double)c * w;
    cnt += c;
    mass += cw;
    if (!(w < min_p)) mass_mp += cw;
  }
  unsigned total_cnt, cnt_upto;
  double total, upto, total_mp, mp_upto;
  const unsigned cnt_before = block_before<unsigned>(cnt, wcnt, cnt_upto, total_cnt, [](unsigned v, int o) { return (unsigned)__shfl_up((int)v, o, 64); });
  const double before = block_before<double>(mass, wsum, upto, total, shfl_up_d);
  (void)block_before<double>(mass_mp, wsum, mp_upto, total_mp, shfl_up_d);
  // top-k: the sum of the first `limit`
  double Z = total;
  if (limit < total_cnt) {
    if (cnt_before < limit && limit <= cnt_upto) {
      unsigned long long left = limit - cnt_before;
      double run = before;
      for (int i = i0; i < i0 + kBpt && left; ++i) {
        const unsigned long long c = min((unsigned long long)hist[i], left);
        if (c) run += (double)c * weight(i);
        left -= c;
      }
      shared_mass = run;
    }
    __syncthreads();
    Z = shared_mass;
  }
  // top-p: the shortest prefix that reaches p * Z
  if (top_p < 1.0) {
    const double goal = top_p * Z;
    __syncthreads();
    if (tid == 0) shared_mass = 1.0;                // at least the first token
    __syncthreads();
    if (before < goal && goal <= upto) {
      double run = before, kept = 1.0;
      for (int i = i0; i < i0 + kBpt; ++i) {
        const unsigned c = hist[i];
        if (!c) continue;
        if (!(run < goal)) break;
        const double w = weight(i);
        const double n = w > 0.0 ? fmin(fmax(ceil((goal - run) / w), 1.0), (double)c) : (double)c;
        kept = run + n * w;
        run += (double)c * w;
      }
      shared_mass = kept;
    }
    __syncthreads();
    Z = fmin(Z, shared_mass);
  }
  Z = fmin(Z, min_p > 1.0 ? 1.0 : total_mp);
  // the first token whose running sum exceeds u * Z
  const float uf = a.u[b];
  const double target = fmin(fmax((double)uf, 0.0), 1.0 - 0x1p-24) * Z;
  if (tid == 0) { pick_bin = 0; pick_rank = 0; }
  __syncthreads();
  if (before <= target && target < upto) {
    double run = before;
    int bin = 0;
    double at = 0.0, w = 1.0;
    unsigned c = 0;
    for (int i = i0; i < i0 + kBpt; ++i) {
      if (!hist[i]) continue;
      const double wi = weight(i);
      if (!(wi > 0.0)) break;
      bin = i; at = run; w = wi; c = hist[i];
      run += (double)c * wi;
      if (run > target) break;
    }
    pick_bin = bin;
    pick_rank = (int)fmin(fmax(floor((target - at) / w), 0.0), (double)(c - 1));
  }
  __syncthreads();
  const int bin = top + pick_bin;
  int rank = pick_rank;
  if (tid == 0) a.logprobs[b] = (float)(log(weight(pick_bin)) - log(Z));
  // the rank-th token (by index) of that value
  for (long long part = 0; part < a.V; part += kRound) {
    if (!resident) x.load(a, row, part, tid);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      unsigned n = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) n += __popcll(__ballot(x.place(c, e) == bin));
      if (lane == 0) matches[c * kWaves + wave] = n;
    }
    __syncthreads();
    int seen = 0, where = -1;
    for (int i = 0; i < kChunks * kWaves; ++i) {
      const int n = (int)matches[i];
      if (where < 0 && rank < seen + n) { where = i; rank -= seen; }
      seen += n;
    }
    if (where >= 0) {
      if (where % kWaves == wave) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          if (c == where / kWaves) {
            int n = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) n += x.place(c, e) == bin;
            int ex = n;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
              const int y = __shfl_up(ex, o, 64);
              if (lane >= o) ex += y;
            }
            ex -= n;
            if (rank >= ex && rank < ex + n) {
              int left = rank - ex;
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (x.place(c, e) == bin && left-- == 0) a.tokens[b] = part + (long long)(c * kThreads + tid) * 8 + e;
            }
          }
      }
      return;
    }
    rank -= seen;
    __syncthreads();
  }
}

}  // namespace

extern "C" int zk_sample(const void* logits, const float* u, const float* temperature_rows, const int32_t* top_k_rows,
                         const float* top_p_rows, const float* min_p_rows, float temperature, int top_k, float top_p,
                         float min_p, int64_t* tokens, float* logprobs, int64_t rows, int64_t V, int64_t ld,
                         hipStream_t stream) {
  if (rows < 0 || rows > 0x7FFFFFFF || V <= 0 || V > 0x7FFFFFFF || ld < V) return ZK_EINVAL;
  if (!logits || !u || !tokens || !logprobs || (reinterpret_cast<uintptr_t>(logits) & 1)) return ZK_EINVAL;
  // settings of the whole call: a number is asked for (NaN is not), top_p and min_p are shares
  if (!temperature_rows && !(temperature >= 0.f && temperature <= kMaxTemperature)) return ZK_EINVAL;
  if (!top_p_rows && !(top_p > 0.f && top_p <= 1.f)) return ZK_EINVAL;
  if (!min_p_rows && !(min_p >= 0.f && min_p <= 1.f)) return ZK_EINVAL;
  if (!top_k_rows && top_k < 0) return ZK_EINVAL;
  if (rows == 0) return ZK_OK;
  SampleArgs a{(const bf16_t*)logits, u, temperature_rows, top_p_rows, min_p_rows, top_k_rows, temperature, top_p, min_p,
               top_k, (long long*)tokens, logprobs, (long long)V, (long long)ld,
               !(reinterpret_cast<uintptr_t>(logits) & 15) && (rows == 1 || !(ld & 7))};
  hipLaunchKernelGGL(sample_kernel, dim3((unsigned)rows), dim3(kThreads), 0, stream, a);
  ZK_CHECK_LAUNCH();
  return ZK_OK;
}
