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
// A thread owns 8 consecutive bins of each of 5 blocks of 8192 (occupied bins come in runs of a few thousand: a thread with
// 39 consecutive ones would form most exponentials alone).
constexpr int kRun = 8, kBlocks = 5, kBlock = kThreads * kRun, kBins = 39936;
constexpr int kChunks = 16;                         // 16-byte chunks of the row a thread holds in registers
constexpr int kRound = kThreads * 8 * kChunks;      // tokens of one register-held part of a row
constexpr float kMaxTemperature = 1048576.0f;
constexpr double kNothing = -64.0;                  // e^-64 of the largest weight: 2^31 such tokens do not move a 64-bit sum

struct SampleArgs {
  const bf16_t* logits;
  const float *u, *temperature_rows, *top_p_rows, *min_p_rows;
  const int* top_k_rows;
  float temperature, top_p, min_p;
  int top_k;
  long long* tokens;
  float* logprobs;
  long long V, ld;
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
  // chunk c of the part: tokens part + (c * kThreads + tid) * 8 - skew .., where skew makes the address 16-byte aligned
  __device__ __forceinline__ void load(const bf16_t* row, long long V, long long part, int skew, int tid) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const long long i = part + (long long)(c * kThreads + tid) * 8 - skew;
      u32x4 x = {0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u};     // -inf outside the row
      if (i >= 0 && i + 8 <= V) {
        x = *reinterpret_cast<const u32x4*>(row + i);
      } else if (i + 8 > 0 && i < V) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e >= 0 && i + e < V) {
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

// inclusive sum over the wave's lanes in DPP steps (rows of 16, then their ends broadcast): no LDS round trips
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp0(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true); }
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp0(double v) {
  return __hiloint2double(dpp0<CTRL, ROWS>(__double2hiint(v)), dpp0<CTRL, ROWS>(__double2loint(v)));
}
template <class T>
__device__ __forceinline__ T wave_upto(T v) {
  v += dpp0<0x111, 0xF>(v);
  v += dpp0<0x112, 0xF>(v);
  v += dpp0<0x114, 0xF>(v);
  v += dpp0<0x118, 0xF>(v);
  v += dpp0<0x142, 0xA>(v);
  v += dpp0<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ double from_lane(double v, int lane) {
  return __hiloint2double(__shfl(__double2hiint(v), lane, 64), __shfl(__double2loint(v), lane, 64));
}
__device__ __forceinline__ int from_lane(int v, int lane) { return __shfl(v, lane, 64); }

// Sums over the bins in order (block, thread) of each thread's five: before[j] = all earlier ones, upto[j] = with this one
// (the same bits as the next one's `before`, so exactly one holds a border); returns the total.  Fixed order.
template <class T>
__device__ __forceinline__ T running(const T (&v)[kBlocks], T (&before)[kBlocks], T (&upto)[kBlocks], T* ends) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) {
    upto[j] = wave_upto(v[j]);
    if (lane == 63) ends[j * kWaves + wave] = upto[j];
  }
  __syncthreads();
  // ends[0 .. 79] -> their own running sums, in every wave by itself
  const T e0 = wave_upto(ends[lane]);
  const T t0 = from_lane(e0, 63);
  const T e1 = wave_upto(lane < kBlocks * kWaves - 64 ? ends[64 + lane] : T(0)) + t0;
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) {
    const int at = j * kWaves + wave - 1;           // the wave before, in order
    const T base = at < 0 ? T(0) : at < 64 ? from_lane(e0, at) : from_lane(e1, at - 64);
    const T prev = from_lane(upto[j], lane ? lane - 1 : 0);
    before[j] = base + (lane ? prev : T(0));
    upto[j] = lane == 63 ? (at + 1 < 64 ? from_lane(e0, at + 1) : from_lane(e1, at + 1 - 64)) : base + upto[j];
  }
  return from_lane(e1, kBlocks * kWaves - 64 - 1);
}

__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned hist[kBins];
  __shared__ double ends_d[kBlocks * kWaves], hit_mass;
  __shared__ int ends_i[kBlocks * kWaves], wtop[kWaves], wnan[kWaves], hit, hit_count;
  __shared__ __attribute__((aligned(16))) unsigned matches[kChunks * kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long b = blockIdx.x;
  const bf16_t* row = a.logits + b * a.ld;
  const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) >> 1);
  const long long span = a.V + skew;
  Row x;
  const bool resident = span <= kRound;
  if (resident) x.load(row, a.V, 0, skew, tid);
  float Tf = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
  const int top_k = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
  const double top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
  const double min_p = a.min_p_rows ? a.min_p_rows[b] : a.min_p;
  const bool first_only = !(Tf > 0.f) || top_k == 1;      // the largest logit: nothing to count
  Tf = fminf(Tf, kMaxTemperature);
  if (!first_only)
    for (int i = tid; i < kBins / 4; i += kThreads) reinterpret_cast<u32x4*>(hist)[i] = u32x4{0u, 0u, 0u, 0u};
  // the largest logit, and whether any is NaN
  int top = kBottom, low = kTop;
  for (long long part = 0; part < span; part += kRound) {
    if (!resident) x.load(row, a.V, part, skew, tid);
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = x.place(c, e);
        top = min(top, d);
        low = max(low, d);
      }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { top = min(top, __shfl_xor(top, o, 64)); low = max(low, __shfl_xor(low, o, 64)); }
  if (lane == 0) { wtop[wave] = top; wnan[wave] = low; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) { top = min(top, wtop[w]); low = max(low, wnan[w]); }
  const bool nan = top < kTop || low > kBottom;
  if (nan || top >= kBottom) {                      // a NaN, or no token that can be drawn
    if (tid == 0) {
      a.tokens[b] = -1;
      a.logprobs[b] = nan ? __builtin_nanf("") : -INFINITY;
    }
    return;
  }
  int bin = 0, rank = 0;
  double logp = 0.0;
  if (!first_only) {
    for (long long part = 0; part < span; part += kRound) {
      if (!resident) x.load(row, a.V, part, skew, tid);
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = x.place(c, e) - top;
          if (d < kBins && d < kBottom - top) atomicAdd(&hist[d], 1u);
        }
    }
    __syncthreads();
    // weight of bin i (a maximum of +inf has the only weight)
    const double vtop = value_of(top), inv_t = 1.0 / (double)Tf;
    auto weight = [&](int i) {
      const double z = (value_of(top + i) - vtop) * inv_t;
      return i == 0 ? 1.0 : z > kNothing ? exp(z) : 0.0;
    };
    int cnt[kBlocks];
    double mass[kBlocks], mass_mp = 0.0;
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) {
      cnt[j] = 0;
      mass[j] = 0.0;
      const int i0 = j * kBlock + tid * kRun;
      if (i0 >= kBins) continue;
      const u32x4 h0 = *reinterpret_cast<const u32x4*>(&hist[i0]), h1 = *reinterpret_cast<const u32x4*>(&hist[i0 + 4]);
      if (!(h0[0] | h0[1] | h0[2] | h0[3] | h1[0] | h1[1] | h1[2] | h1[3])) continue;
#pragma unroll 1
      for (int i = i0; i < i0 + kRun; ++i) {
        const int c = (int)hist[i];
        if (!c) continue;
        const double w = weight(i), cw = (double)c * w;
        cnt[j] += c;
        mass[j] += cw;
        if (!(w < min_p)) mass_mp += cw;
      }
    }
    double before[kBlocks], upto[kBlocks];
    const double total = running(mass, before, upto, ends_d);
    double Z = total;
    // one thread's eight bins, on lanes 0 .. 7 of every wave: count, weight, and the sum before each from `from` on
    int c8;
    double w8, run8;
    auto spread = [&](int at, double from) {
      const int i = at * kRun + (lane & 7);       // thread t of block j: at = j * kThreads + t
      c8 = (int)hist[i];
      w8 = c8 ? weight(i) : 0.0;
      double v = (double)c8 * w8;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const double y = from_lane(v, lane >= o ? lane - o : 0);
        if ((lane & 7) >= o) v += y;
      }
      run8 = from + v - (double)c8 * w8;
    };
    // the first eight bins, in order, that hold weight and whose running sum passes a border
    auto find = [&](auto passes) {
      if (tid == 0) hit = 0x7FFFFFFF;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        const unsigned long long any = __ballot(mass[j] > 0.0 && passes(upto[j]));
        if (any && lane == __ffsll(any) - 1) atomicMin(&hit, j * kThreads + tid);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kBlocks; ++j)
        if (hit == j * kThreads + tid) hit_mass = before[j];
      __syncthreads();
      spread(hit, hit_mass);
    };
    // top-k: the sum of the first top_k
    if (top_k > 0) {
      int cnt_before[kBlocks], cnt_upto[kBlocks];
      if (running(cnt, cnt_before, cnt_upto, ends_i) > top_k) {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j)
          if (cnt_before[j] < top_k && top_k <= cnt_upto[j]) { hit = j * kThreads + tid; hit_count = cnt_before[j]; hit_mass = before[j]; }
        __syncthreads();
        spread(hit, hit_mass);
        int n = c8;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
          const int y = from_lane(n, lane >= o ? lane - o : 0);
          if ((lane & 7) >= o) n += y;
        }
        const int left = top_k - (hit_count + n - c8);     // of this bin and later ones
        const int last = __ffsll(__ballot(lane < 8 && left <= c8 && c8 > 0)) - 1;
        Z = from_lane(run8 + (double)min(max(left, 0), c8) * w8, last < 0 ? 7 : last);
        __syncthreads();
      }
    }
    // top-p: the shortest prefix that reaches p * Z
    if (top_p < 1.0) {
      const double goal = top_p * Z;
      find([&](double sum) { return sum >= goal; });
      const unsigned long long full = __ballot(lane < 8 && w8 > 0.0);
      const unsigned long long over = __ballot(lane < 8 && w8 > 0.0 && run8 + (double)c8 * w8 >= goal);
      const int e = over ? __ffsll(over) - 1 : 63 - __clzll(full);
      const double n = fmin(fmax(ceil((goal - run8) / w8), 1.0), (double)c8);
      Z = fmin(Z, from_lane(run8 + n * w8, e));
      __syncthreads();
    }
    if (min_p > 0.0) {
      const double s = wave_upto(mass_mp);
      __syncthreads();                              // the running sums' ends have been read
      if (lane == 63) ends_d[wave] = s;
      __syncthreads();
      double mp = 0.0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) mp += ends_d[w];
      Z = fmin(Z, min_p > 1.0 ? 1.0 : mp);
    }
    // the first token whose running sum exceeds u * Z
    const double target = fmin(fmax((double)a.u[b], 0.0), 1.0 - 0x1p-24) * Z;
    find([&](double sum) { return sum > target; });
    const unsigned long long full = __ballot(lane < 8 && w8 > 0.0);
    const unsigned long long over = __ballot(lane < 8 && w8 > 0.0 && run8 + (double)c8 * w8 > target);
    const int e = over ? __ffsll(over) - 1 : 63 - __clzll(full);
    bin = hit * kRun + e;
    rank = (int)from_lane(fmin(fmax(floor((target - run8) / w8), 0.0), (double)(c8 - 1)), e);
    const double w = from_lane(w8, e);
    if (tid == 0) logp = log(w) - log(Z);
  }
  if (tid == 0) a.logprobs[b] = (float)logp;
  bin += top;
  // the rank-th token (by index) of that value
  for (long long part = 0; part < span; part += kRound) {
    if (!resident) x.load(row, a.V, part, skew, tid);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      unsigned n = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) n += __popcll(__ballot(x.place(c, e) == bin));
      if (lane == 0) matches[c * kWaves + wave] = n;
    }
    __syncthreads();
    const u32x4 m4 = *reinterpret_cast<const u32x4*>(&matches[lane * 4]);
    const int mine = (int)(m4[0] + m4[1] + m4[2] + m4[3]);
    const int end = wave_upto(mine), start = end - mine;
    const unsigned long long has = __ballot(rank >= start && rank < end);
    if (has) {
      int where = lane * 4, left = rank - start;
#pragma unroll
      for (int q = 0; q < 3; ++q)
        if (where == lane * 4 + q && left >= (int)m4[q]) { left -= (int)m4[q]; ++where; }
      const int owner = __ffsll(has) - 1;
      where = from_lane(where, owner);
      left = from_lane(left, owner);
      if (where % kWaves == wave) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          if (c == where / kWaves) {
            int n = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) n += x.place(c, e) == bin;
            const int ex = wave_upto(n) - n;
            if (left >= ex && left < ex + n) {
              int k = left - ex;
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (x.place(c, e) == bin && k-- == 0) a.tokens[b] = part + (long long)(c * kThreads + tid) * 8 - skew + e;
            }
          }
      }
      return;
    }
    rank -= from_lane(end, 63);
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
               top_k, (long long*)tokens, logprobs, (long long)V, (long long)ld};
  hipLaunchKernelGGL(sample_kernel, dim3((unsigned)rows), dim3(kThreads), 0, stream, a);
  ZK_CHECK_LAUNCH();
  return ZK_OK;
}
