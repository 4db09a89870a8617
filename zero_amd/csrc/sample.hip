// Drawing the next token of every row of bf16 logits: temperature, top-k, top-p, min-p, from a given number u.
//
// Definition (per row).  Tokens in falling order of their logit, equal logits by the lower index; w_r = e^((l_r - max) / T).
//   top-k keeps the first k; top-p the shortest prefix whose sum reaches p times the sum of what top-k kept; min-p the
//   tokens with w >= min_p.  All three are prefixes of one order, so the kept set is the shortest of them, and the token
//   drawn is the first whose running sum exceeds u * Z, Z = the kept sum.  logprob = log(w / Z).
//
// bf16 logits have at most 65 281 different values that can be drawn, so the sorted row is its HISTOGRAM: bins in
// falling order of the value hold how many tokens have it, a bin of c tokens adds c * w to the running sum, and no sort
// of 10^5 tokens is needed.  One workgroup owns a row; its bins live in LDS as 32-bit counts (see HALF).  Sums are formed in
// 64 bits over the occupied bins only (a few thousand exponentials instead of one per token), so that the token does not
// depend on how a sum was split: the running sum of 10^5 weights in 32 bits would move its borders by more than the
// weight of a rare token.
//
// 39 936 bins (156 KiB of the CU's 160) instead of 65 281: bin 0 is up to 512 values above the maximum, so a token below the
// last bin is more than 39 423 values below the maximum.  Two bf16 of one sign are at most 32 640 values apart, so the
// signs differ and one of the two magnitudes is beyond 2^27: weight e^-128 at 2^20, the largest temperature used, which
// moves no sum of 2^31 weights in 64 bits.
//
// 128 256 tokens of one row: 21.1 us, 50 thousand clocks, of which the first tokens' way takes 6, the 128 256 LDS counts 20
// (10 a wave of 64, bank conflicts of random bins), the weights 6, running sums 3, borders 4 each, the search for the token
// 4.  512 rows of 128 256 (131 MB): 55 us, two rounds of 256 workgroups; 156 KiB of bins leave a CU to one row, so that no
// other row's work fills these waits.  61 rows of 32 003: 15.3 us.
#include "common.h"
#include "../../include/zero_hip.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
// A thread owns 8 consecutive bins of each of 5 blocks of 8192 (occupied bins come in runs of a few thousand: a thread with
// 39 consecutive ones would form most exponentials alone).
constexpr int kRun = 8, kBlocks = 5, kBlock = kThreads * kRun, kBins = 39936;
constexpr int kChunks = 16;                         // 16-byte chunks of the row a thread holds in registers, at most
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

// A logit's key: its sign-magnitude bits as a two's complement number, so that keys are in the logits' order and -0 is +0.
// +inf 0x7F80, -inf -0x7F80, beyond these: NaN.  Two keys to a register, as the logits come: packed 16-bit instructions
// make them, find the largest and count matches, at one to two instructions a token (a single workgroup has one CU for 10^5
// tokens: every instruction per token is 0.7 us).
typedef __attribute__((ext_vector_type(2))) short s16x2;
constexpr int kInf = 0x7F80;
constexpr int kAbove = 512;
__device__ __forceinline__ unsigned keys_of(unsigned w) {
  const s16x2 m = __builtin_bit_cast(s16x2, w) >> (s16x2)15;
  return __builtin_bit_cast(unsigned, (s16x2)((__builtin_bit_cast(s16x2, w & 0x7FFF7FFFu) ^ m) - m));
}
__device__ __forceinline__ double value_of(int key) {
  return (double)bf2f((bf16_t)(key < 0 ? 0x8000u | (unsigned)-key : (unsigned)key));
}

// e^z for z in (-64, 0]: z = n ln 2 + r with |r| <= ln 2 / 2, the Taylor series of e^r up to r^13 / 13! (what is left out is
// 4e-18 of it), its halves side by side, and n added to the exponent.  Off by about one step of 2^-52; no special cases.
__device__ __forceinline__ double exp_of(double z) {
  const double n = rint(z * 1.4426950408889634);
  double r = fma(n, -0x1.62e42fefa38p-1, z);        // ln 2 in two parts, the first with zeros behind it: n times it is exact
  r = fma(n, -0x1.ef35793c7673p-45, r);
  const double r2 = r * r, r4 = r2 * r2;
  const double a = fma(fma(r, 1.0 / 6, 0.5), r2, 1.0 + r);
  const double b = fma(fma(r, 1.0 / 5040, 1.0 / 720), r2, fma(r, 1.0 / 120, 1.0 / 24));
  const double c = fma(fma(r, 1.0 / 39916800, 1.0 / 3628800), r2, fma(r, 1.0 / 362880, 1.0 / 40320));
  const double d = fma(r, 1.0 / 6227020800.0, 1.0 / 479001600);
  const double y = fma(fma(fma(d, r4, c), r4, b), r4, a);
  return __hiloint2double(__double2hiint(y) + ((int)n << 20), __double2loint(y));
}

typedef u32x4 u32x4_any __attribute__((aligned(2)));          // rows start at any token: 16-byte loads from 2-byte addresses

// A part of a row in registers: chunk c of thread tid is tokens (c * kThreads + tid) * 8 .. of it, at p.  Chunks that the row
// ends in or before are the last 8 tokens (so that every load is alike, and nothing waits for one early); what of them the
// chunks before hold too becomes -inf with the keys.
template <int NC>
struct Row {
  u32x4 r[NC];
  // n: tokens left from p on; at least 8 tokens up to p + n.  No branch: a wait for one chunk then leaves the later ones in
  // flight.
  __device__ __forceinline__ void load(const bf16_t* p, int n, int tid) {
#pragma unroll
    for (int c = 0; c < NC; ++c) r[c] = *reinterpret_cast<const u32x4_any*>(p + min((c * kThreads + tid) * 8, n - 8));
  }
  __device__ __forceinline__ void none(int c) { r[c] = u32x4{0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u}; }   // -inf
  // the same for a row of fewer than 8 tokens, so placed that its end is the chunk's
  __device__ __forceinline__ void load_short(const bf16_t* p, int n, int tid) {
#pragma unroll
    for (int c = 0; c < NC; ++c) none(c);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e >= 8 - n) {
        const unsigned v = p[e - (8 - n)];
        r[0][e >> 1] = e & 1 ? (r[0][e >> 1] & 0xFFFFu) | (v << 16) : (r[0][e >> 1] & 0xFFFF0000u) | v;
      }
  }
  __device__ __forceinline__ void to_keys(int c, int n, int tid) {
    const int s = (c * kThreads + tid) * 8 + 8 - n;
    if (s > 0) {                                    // the first s tokens are other chunks'
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned w = r[c][e];
        r[c][e] = s > 2 * e + 1 ? 0xFF80FF80u : s > 2 * e ? (w & 0xFFFF0000u) | 0xFF80u : w;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) r[c][e] = keys_of(r[c][e]);
  }
};

__device__ __forceinline__ double lane_of(double v, int lane) {     // lane: the same in the whole wave
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Sums over the bins in order (block, thread) of each thread's five: before[j] = all earlier ones, upto[j] = with this one;
// returns the total.  Fixed order.
template <class T>
__device__ __forceinline__ T running(const T (&v)[kBlocks], T (&before)[kBlocks], T (&upto)[kBlocks], T* ends) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) {
    upto[j] = __any(v[j] != T(0)) ? wave_upto(v[j]) : T(0);     // (most waves' bins of a block are empty)
    if (lane == 63) ends[j * kWaves + wave] = upto[j];
  }
  __syncthreads();
  // ends[0 .. 79] -> their own running sums, in every wave by itself
  const T e0 = wave_upto(ends[lane]);
  const T e1 = wave_upto(lane < kBlocks * kWaves - 64 ? ends[64 + lane] : T(0)) + lane_of(e0, 63);
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) {
    const int at = j * kWaves + wave - 1;           // the wave before, in order
    const T base = at < 0 ? T(0) : at < 64 ? lane_of(e0, at & 63) : lane_of(e1, at & 63);
    before[j] = base + dpp0<0x138, 0xF>(upto[j]);   // the lane before; lane 0: nothing
    upto[j] = base + upto[j];
  }
  return lane_of(e1, kBlocks * kWaves - 64 - 1);
}

__device__ __forceinline__ void sync_lds() {       // a barrier for LDS alone: loads in flight stay in flight
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// RESIDENT: the row (8 tokens or more) fits NC chunks a thread (131 072 tokens at most) and is read once; otherwise each pass
// over the row reads it again, part by part.
// HALF: the bins are 16 bits wide (rows of up to 32 768 tokens).
// The counting does not wait for the row: as soon as the first 8192 tokens are there, bin 0 is put 512 values (a factor of
// 16) above the largest of them, and every chunk is counted as it arrives (1 x 128256: 23.7 -> 22.0 us, 512 x 128256: 60.4 ->
// 57.1, against counting once the maximum is known).  If a later token is above bin 0 after all, the counts are cleared and
// made again from the true maximum.
template <int NC, bool RESIDENT, bool HALF>
__global__ __launch_bounds__(kThreads, HALF ? 8 : 4) void sample_kernel(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned hist[HALF ? kBins / 2 : kBins];
  auto counted = [&](int i) { return HALF ? (int)reinterpret_cast<const unsigned short*>(hist)[i] : (int)hist[i]; };
  __shared__ double ends_d[kBlocks * kWaves], mp_d[kWaves], cand_mass[3][kWaves], kept[3];
  __shared__ int ends_i[kBlocks * kWaves], cand[3][kWaves], cand_count[kWaves], wtop[kWaves], wlow[kWaves], first[kWaves], picked[2];
  unsigned* matches = hist;                         // [kChunks * kWaves], once the counts are done with
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long b = blockIdx.x, V = a.V;
  const bf16_t* row = a.logits + b * a.ld;
  auto left = [&](long long part) { return RESIDENT ? (int)V : (int)min(V - part, (long long)kRound); };
  Row<NC> x;
  auto read = [&](long long part) {
    if (V >= 8) x.load(row + part, left(part), tid);
    else x.load_short(row, (int)V, tid);
  };
  if (RESIDENT) x.load(row, left(0), tid);
  float Tf = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
  const int top_k = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
  const double top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
  const double min_p = a.min_p_rows ? a.min_p_rows[b] : a.min_p;
  const float u = a.u[b];
  const bool first_only = !(Tf > 0.f) || top_k == 1;      // the largest logit: nothing to count
  Tf = fminf(Tf, kMaxTemperature);
  auto clear = [&]() {
    for (int i = tid; i < kBins / (HALF ? 8 : 4); i += kThreads) reinterpret_cast<u32x4*>(hist)[i] = u32x4{0u, 0u, 0u, 0u};
  };
  int base = 0;                                     // the key of bin 0
  // bin d counts the tokens of key base - d (its byte offset is one multiply-add; -inf has no weight)
  constexpr int BB = HALF ? 2 : 4;                  // bytes a bin
  auto count = [&](const u32x4& keys) {
    const int base_b = base * BB, base16 = base * 16;
    auto add = [&](unsigned d, unsigned d16) __attribute__((always_inline)) {
      if (d < (unsigned)kBins * BB)                 // (half: 16 d is 0 or 16 in the five bits of a shift)
        atomicAdd(reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(hist) + (HALF ? d & ~3u : d)), HALF ? 1u << (d16 & 31) : 1u);
    };
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned w = keys[e];
      unsigned d0, d1, s0 = 0, s1 = 0;
      asm("v_mad_i32_i16 %0, %1, %2, %3" : "=v"(d0) : "v"(w), "v"(-BB), "v"(base_b));
      asm("v_mad_i32_i16 %0, %1, %2, %3 op_sel:[1,0,0,0]" : "=v"(d1) : "v"(w), "v"(-BB), "v"(base_b));
      if (HALF) {
        asm("v_mad_i32_i16 %0, %1, %2, %3" : "=v"(s0) : "v"(w), "v"(-16), "v"(base16));
        asm("v_mad_i32_i16 %0, %1, %2, %3 op_sel:[1,0,0,0]" : "=v"(s1) : "v"(w), "v"(-16), "v"(base16));
      }
      add(d0, s0);
      add(d1, s1);
    }
  };
  if (!first_only) clear();
  // the largest logit, whether any is NaN, and the counts
  s16x2 hi2 = {-32768, -32768}, lo2 = {32767, 32767};
  for (long long part = 0; part < (RESIDENT ? 1 : V); part += kRound) {
    if (!RESIDENT) read(part);
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (c * kThreads * 8 < left(part)) {
        x.to_keys(c, left(part), tid);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned w = x.r[c][e];             // (a bit cast of a vector's element takes the vector's first one)
          hi2 = __builtin_elementwise_max(hi2, __builtin_bit_cast(s16x2, w));
          lo2 = __builtin_elementwise_min(lo2, __builtin_bit_cast(s16x2, w));
        }
        if (!first_only) {
          if (c == 0 && part == 0) {
            int m = max((int)hi2[0], (int)hi2[1]);
            m = wave_top(m);
            if (lane == 0) first[wave] = m;
            sync_lds();
            m = first[lane & (kWaves - 1)];
            m = wave_top(m);
            base = __builtin_amdgcn_readfirstlane(min(m + kAbove, kInf));
          }
          count(x.r[c]);
        }
      } else {
        x.none(c);
      }
  }
  int top = wave_top(max((int)hi2[0], (int)hi2[1])), low = -wave_top(-min((int)lo2[0], (int)lo2[1]));
  if (lane == 0) { wtop[wave] = top; wlow[wave] = low; }
  __syncthreads();
  top = wave_top(wtop[lane & (kWaves - 1)]);
  low = -wave_top(-wlow[lane & (kWaves - 1)]);
  const bool nan = top > kInf || low < -kInf;
  if (nan || top == -kInf) {                        // a NaN, or no token that can be drawn
    if (tid == 0) {
      a.tokens[b] = -1;
      a.logprobs[b] = nan ? __builtin_nanf("") : -INFINITY;
    }
    return;
  }
  top = __builtin_amdgcn_readfirstlane(top);
  int bin = 0, rank = 0;
  if (!first_only) {
    if (top > base) {                               // (uniform)
      clear();
      base = top;
      __syncthreads();
      for (long long part = 0; part < (RESIDENT ? 1 : V); part += kRound) {
        if (!RESIDENT) read(part);
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (c * kThreads * 8 < left(part)) {
            if (!RESIDENT) x.to_keys(c, left(part), tid);
            count(x.r[c]);
          }
      }
      __syncthreads();
    }
    // weight of bin i (a maximum of +inf has the only weight; the bins above the maximum are empty)
    const double vtop = value_of(top), inv_t = 1.0 / (double)Tf;
    auto weight = [&](int i) {
      const double z = (value_of(base - i) - vtop) * inv_t;
      return i == base - top ? 1.0 : z > kNothing ? exp_of(z) : 0.0;
    };
    int cnt[kBlocks];
    double mass[kBlocks], mass_mp = 0.0;
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) {
      cnt[j] = 0;
      mass[j] = 0.0;
      const int i0 = j * kBlock + tid * kRun;
      if (i0 >= kBins) continue;
      u32x4 any = *reinterpret_cast<const u32x4*>(&hist[HALF ? i0 / 2 : i0]);
      if (!HALF) any |= *reinterpret_cast<const u32x4*>(&hist[i0 + 4]);
      if (!(any[0] | any[1] | any[2] | any[3])) continue;
      int c_next = counted(i0);
#pragma unroll 1
      for (int i = i0; i < i0 + kRun; ++i) {
        const int c = c_next;
        c_next = counted(min(i + 1, kBins - 1));
        if (!c) continue;
        const double w = weight(i), cw = (double)c * w;
        cnt[j] += c;
        mass[j] += cw;
        if (!(w < min_p)) mass_mp += cw;
      }
    }
    mass_mp = wave_upto(mass_mp);
    if (lane == 63) mp_d[wave] = mass_mp;
    double before[kBlocks], upto[kBlocks];
    const double total = running(mass, before, upto, ends_d);
    double Z = total;
    // Borders.  Each wave names its first eight bins, in order, that hold weight and whose running sum passes the border;
    // the first of these resolves it: its bins on lanes 0 .. 7 of wave 0, count, weight and running sum each.
    int c8 = 0;
    double w8 = 0.0, run8 = 0.0;
    auto spread = [&](int at, double from) {
      const int i = at * kRun + (lane & 7);         // thread t of block j: at = j * kThreads + t
      c8 = counted(i);
      w8 = c8 ? weight(i) : 0.0;
      double v = (double)c8 * w8;
      v += dpp0<0x111, 0xF>(v) * (double)((lane & 7) >= 1);
      v += dpp0<0x112, 0xF>(v) * (double)((lane & 7) >= 2);
      v += dpp0<0x114, 0xF>(v) * (double)((lane & 7) >= 4);
      run8 = from + v - (double)c8 * w8;
    };
    auto find = [&](int k, auto passes) {           // -> which eight bins, in wave 0
#pragma unroll
      for (int j = kBlocks - 1; j >= 0; --j) {
        const unsigned long long any = __ballot(mass[j] > 0.0 && passes(upto[j]));
        if (j == kBlocks - 1 && lane == 0) cand[k][wave] = 0x7FFFFFFF;
        if (any && lane == __ffsll(any) - 1) { cand[k][wave] = j * kThreads + tid; cand_mass[k][wave] = before[j]; }
      }
      __syncthreads();
      int at = 0;
      if (wave == 0) {
        const int mine = lane < kWaves ? cand[k][lane] : 0x7FFFFFFF;
        at = -wave_top(-mine);
        spread(at, cand_mass[k][__ffsll(__ballot(mine == at)) - 1]);
      }
      return at;
    };
    // top-k: the sum of the first top_k
    if (top_k > 0) {
      int cnt_before[kBlocks], cnt_upto[kBlocks];
      if (running(cnt, cnt_before, cnt_upto, ends_i) > top_k) {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j)
          if (cnt_before[j] < top_k && top_k <= cnt_upto[j]) { cand[0][0] = j * kThreads + tid; cand_count[0] = cnt_before[j]; cand_mass[0][0] = before[j]; }
        __syncthreads();
        if (wave == 0) {
          spread(cand[0][0], cand_mass[0][0]);
          int n = c8;
          n += dpp0<0x111, 0xF>(n) * (int)((lane & 7) >= 1);
          n += dpp0<0x112, 0xF>(n) * (int)((lane & 7) >= 2);
          n += dpp0<0x114, 0xF>(n) * (int)((lane & 7) >= 4);
          const int k = top_k - (cand_count[0] + n - c8);     // of this bin and later ones
          if (lane == __ffsll(__ballot(lane < 8 && c8 > 0 && k <= c8)) - 1) kept[0] = run8 + (double)k * w8;
        }
        __syncthreads();
        Z = kept[0];
      }
    }
    // top-p: the shortest prefix that reaches p * Z
    if (top_p < 1.0) {
      const double goal = top_p * Z;
      find(1, [&](double sum) { return sum >= goal; });
      if (wave == 0) {
        const unsigned long long full = __ballot(lane < 8 && w8 > 0.0);
        const unsigned long long over = __ballot(lane < 8 && w8 > 0.0 && run8 + (double)c8 * w8 >= goal);
        const double n = fmin(fmax(ceil((goal - run8) / w8), 1.0), (double)c8);
        if (lane == (over ? __ffsll(over) - 1 : 63 - __clzll(full))) kept[1] = run8 + n * w8;
      }
      __syncthreads();
      Z = fmin(Z, kept[1]);
    }
    if (min_p > 0.0) {
      double mp = 0.0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) mp += mp_d[w];
      Z = fmin(Z, min_p > 1.0 ? 1.0 : mp);
    }
    // the first token whose running sum exceeds u * Z
    const double target = fmin(fmax((double)u, 0.0), 1.0 - 0x1p-24) * Z;
    const int at = find(2, [&](double sum) { return sum > target; });
    if (wave == 0) {
      const unsigned long long full = __ballot(lane < 8 && w8 > 0.0);
      const unsigned long long over = __ballot(lane < 8 && w8 > 0.0 && run8 + (double)c8 * w8 > target);
      if (lane == (over ? __ffsll(over) - 1 : 63 - __clzll(full))) {
        picked[0] = at * kRun + lane;
        picked[1] = (int)fmin(fmax(floor((target - run8) / w8), 0.0), (double)(c8 - 1));
        a.logprobs[b] = (float)(log(w8) - log(Z));
      }
    }
    __syncthreads();
    bin = picked[0] - (base - top);                 // from the maximum's on
    rank = picked[1];
  } else if (tid == 0) {
    a.logprobs[b] = 0.f;
  }
  const int key = __builtin_amdgcn_readfirstlane(top - bin);
  const unsigned key2 = ((unsigned)key & 0xFFFFu) * 0x10001u;
  // the rank-th token (by index) of that value
  for (long long part = 0; part < (RESIDENT ? 1 : V); part += kRound) {
    if (!RESIDENT) {
      read(part);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (c * kThreads * 8 < left(part)) x.to_keys(c, left(part), tid);
        else x.none(c);
    }
    typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
#pragma unroll
    for (int c4 = 0; c4 < kChunks; c4 += 4) {       // most groups of chunks hold no match: one test for four
      int mine[4] = {0, 0, 0, 0};
      if (c4 < NC && c4 * kThreads * 8 < left(part)) {
        u16x2 least = {0xFFFF, 0xFFFF};             // of x ^ key: zero in a half that matches
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned w = x.r[(c4 + k) % NC][e] ^ key2;
            least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2, w));
          }
        if (__any(least[0] == 0 || least[1] == 0)) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            u16x2 other = {0, 0};                   // halves that differ: min(x ^ key, 1), one packed instruction in
#pragma unroll                                      // place of the compiler's compare and select for each half
            for (int e = 0; e < 4; ++e) {
              unsigned w;
              asm("v_pk_min_u16 %0, %1, 1 op_sel_hi:[1,0]" : "=v"(w) : "v"(x.r[(c4 + k) % NC][e] ^ key2));
              other += __builtin_bit_cast(u16x2, w);
            }
            const unsigned sum = __builtin_bit_cast(unsigned, other);
            mine[k] = wave_upto(8 - (int)((sum & 0xFFFFu) + (sum >> 16)));
          }
        }
      }
      if (lane == 63) {
#pragma unroll
        for (int k = 0; k < 4; ++k) matches[(c4 + k) * kWaves + wave] = (unsigned)mine[k];
      }
    }
    __syncthreads();
    const u32x4 m4 = *reinterpret_cast<const u32x4*>(&matches[lane * 4]);
    const int mine = (int)(m4[0] + m4[1] + m4[2] + m4[3]);
    const int end = wave_upto(mine), start = end - mine;
    const unsigned long long has = __ballot(rank >= start && rank < end);
    if (has) {
      int where = lane * 4, k = rank - start;
#pragma unroll
      for (int q = 0; q < 3; ++q)
        if (where == lane * 4 + q && k >= (int)m4[q]) { k -= (int)m4[q]; ++where; }
      const int owner = __ffsll(has) - 1;
      where = lane_of(where, owner);
      k = lane_of(k, owner);
      if (where % kWaves == wave) {
        u32x4 y = x.r[0];
#pragma unroll
        for (int c = 1; c < NC; ++c)
          if (c == where / kWaves) y = x.r[c];
        auto hit = [&](int e) { return ((y[e >> 1] ^ key2) & (e & 1 ? 0xFFFF0000u : 0xFFFFu)) == 0; };
        int n = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) n += hit(e);
        const int ex = wave_upto(n) - n;
        if (k >= ex && k < ex + n) {
          int m = k - ex;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (hit(e) && m-- == 0) a.tokens[b] = part + min((where / kWaves * kThreads + tid) * 8, left(part) - 8) + e;
        }
      }
      return;
    }
    rank -= lane_of(end, 63);
    __syncthreads();
  }
}

}  // namespace

extern "C" int zk_sample(const void* logits, const float* u, const float* temperature_rows, const int32_t* top_k_rows,
                         const float* top_p_rows, const float* min_p_rows, float temperature, int top_k, float top_p,
                         float min_p, int64_t* tokens, float* logprobs, int64_t rows, int64_t V, int64_t ld,
                         hipStream_t stream) {
  if (rows < 0 || rows > 0x7FFFFFFF || V <= 0 || V > 0x7FFFFFFF || ld < V) return ZK_EINVAL;
  if (zk_too_many(rows, kThreads)) return ZK_EINVAL;
  if (!logits || !u || !tokens || !logprobs || (reinterpret_cast<uintptr_t>(logits) & 1)) return ZK_EINVAL;
  // settings of the whole call: a number is asked for (NaN is not), top_p and min_p are shares
  if (!temperature_rows && !(temperature >= 0.f && temperature <= kMaxTemperature)) return ZK_EINVAL;
  if (!top_p_rows && !(top_p > 0.f && top_p <= 1.f)) return ZK_EINVAL;
  if (!min_p_rows && !(min_p >= 0.f && min_p <= 1.f)) return ZK_EINVAL;
  if (!top_k_rows && top_k < 0) return ZK_EINVAL;
  if (rows == 0) return ZK_OK;
  SampleArgs a{(const bf16_t*)logits, u, temperature_rows, top_p_rows, min_p_rows, top_k_rows, temperature, top_p, min_p,
               top_k, (long long*)tokens, logprobs, (long long)V, (long long)ld};
  // more rows than CUs, and few enough tokens for counts of 16 bits: 78 KiB of bins, so that two rows share a CU and one works
  // while the other waits (1024 x 300 43 -> 31 us, 512 x 4681 23.9 -> 19.6, 512 x 32003 28.7 -> 26.3; but 256 x 32003 15.0 ->
  // 17.7, on half the registers and with more instructions a count)
  const bool two = rows > 256;
  void (*kern)(SampleArgs) = V < 8 || V > kRound ? sample_kernel<kChunks, false, false>
                             : V > kRound / 4    ? sample_kernel<kChunks, true, false>
                             : two               ? sample_kernel<kChunks / 4, true, true> : sample_kernel<kChunks / 4, true, false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)rows), dim3(kThreads), 0, stream, a);
  ZK_CHECK_LAUNCH();
  return ZK_OK;
}
