// The norm and rotation of queries and keys where a head is not whole runs of channels: any width, pairs and
// alignment, a lane a pair of single channels.
//
// A warp takes an item of up to 32 rows (a row: one head of one token), of several tokens where a token has few
// heads. Each lane first finds one row's addresses; the first batch of rows (U a team) is on its way while all of them
// find the tokens' angles (into shared memory), and each next one while its predecessor is worked on. The sums of a
// batch go through one another: lanes trade halves of the rows at the first steps, so that U sums over a team take
// U - 1 exchanges and a few more instead of five each.
//
// Measured on one B200 (us; in brackets as heads.cu's rings of one token an item did it, with single channels):
//   65536 tokens, 8 + 8 heads x 37 bf16     forward 109 (150), backward 162 (232)
//   65536 tokens, 8 + 8 heads x 151 bf16    forward 254 (334), backward 363 (414)
//   79000 tokens, 2 + 2 heads x 51 fp32     forward 51 (107), backward 68 (137)
//   20000 tokens, 4 + 4 heads x 500 bf16    forward 184 (170), backward 250 (182): no registers are left for a batch
//   500000 tokens, 4 + 4 heads x 32 bf16    forward 234, backward 327 with 15 pairs in halves (16 pairs are whole runs
//                                           and take heads.cu's rings: 130 and 194)
// Bound by instructions: 2-byte loads and stores, and at 37 channels 19 of 32 lanes. Rows staged through shared memory
// by asynchronous copies of the 16 bytes around them instead: 37 channels 125 and 202, 151 298 and 532.
#include <type_traits>

#include "heads.cuh"
#include "launch.cuh"

namespace ffb {
namespace heads {
namespace {

constexpr int kRows = 32;          // an item's at most
constexpr int kItemPairs = 256;    // angles an item holds, at most (or one token's)

// q's or k's items: `tokens` tokens of `heads` heads each (one token where not all heads are in one item).
struct Phase {
  uint32_t items;
  Divisor chunks, row_heads;  // items a token group; heads a row of tokens
  int tokens, heads;
};
struct AnyPlan {
  Phase phase[2];
  Divisor tokens, pairs;
  uint32_t total;           // tokens
  int shift, turns, table;  // log2 of the lanes a team; an item's angles at most; pairs, to a multiple of 4
  bool fits;                // items are numbered in 31 bits
};

// A warp's rows: element offsets in NT inputs and the output, and where their token's angles lie.
template <int NT>
struct Rows {
  int64_t (*offsets)[kRows];  // [NT + 1]
  int64_t* places;            // [kRows]: of the item's tokens' positions
  int* tables;                // [kRows]
  float2* turns;
  int count, tokens;

  static __host__ __device__ int bytes(int turns) { return (NT + 2) * kRows * 8 + kRows * 4 + turns * 8; }
  __device__ __forceinline__ explicit Rows(uint8_t* smem)
      : offsets(reinterpret_cast<int64_t(*)[kRows]>(smem)), places(offsets[NT + 1]), tables(reinterpret_cast<int*>(places + kRows)),
        turns(reinterpret_cast<float2*>(tables + kRows)), count(0), tokens(0) {}
  // an item's rows
  __device__ __forceinline__ void enter(const HeadsParams& p, const AnyPlan& plan, int which, uint32_t id) {
    const Phase& phase = plan.phase[which];
    const RotaryParams& r = p.rotary;
    const int lane = threadIdx.x & 31;
    const uint32_t group = phase.chunks.quotient(id), first = group * phase.tokens;
    const int head0 = static_cast<int>(id - group * phase.chunks.d) * phase.heads;
    tokens = min(static_cast<uint32_t>(phase.tokens), plan.total - first);
    count = tokens * min(phase.heads, p.heads[which] - head0);
    __syncwarp();
    if (lane < count) {
      const uint32_t of = phase.row_heads.quotient(lane);
      const uint32_t b = plan.tokens.quotient(first + of), t = first + of - b * plan.tokens.d;
      const int head = head0 + lane - static_cast<int>(of) * phase.heads;
      const auto at = [&](const HeadView& v) { return b * v.batch + t * v.token + head * v.head; };
      offsets[0][lane] = at(p.x[which]);
      if constexpr (NT == 2) offsets[1][lane] = at(p.dy[which]);
      offsets[NT][lane] = at(p.out[which]);
      tables[lane] = static_cast<int>(of) * r.pairs;
    }
    if (lane < tokens && r.pairs > 0) {
      const uint32_t b = plan.tokens.quotient(first + lane), t = first + lane - b * plan.tokens.d;
      places[lane] = b * r.batch + t * r.token;
    }
    __syncwarp();
  }
  // its tokens' angles
  __device__ __forceinline__ void find_turns(const RotaryParams& r, const AnyPlan& plan, const Constants& constants) {
    for (int e = threadIdx.x & 31; e < tokens * r.pairs; e += 32) {
      const int of = static_cast<int>(plan.pairs.quotient(e)), j = e - of * r.pairs;
      turns[e] = turn_of(position_at(r, places[of] + constants.axes[j] * r.axis) * constants.quarters[j], r.inverse ? 0x80000000u : 0u);
    }
    __syncwarp();
  }
};

// A lane's pair: `slot` numbers the turned pairs first, then the other channels two by two (the last may stand alone).
struct Spot {
  int a, b, pair;
  bool turned, has_a, has_b;
  __device__ __forceinline__ Spot() {}
  __device__ __forceinline__ Spot(const RotaryParams& r, int slot, int channels) : pair(slot), turned(slot < r.pairs) {
    const bool halves = turned && !r.interleaved;
    a = halves ? slot : 2 * slot;
    b = halves ? r.pairs + slot : 2 * slot + 1;
    has_a = a < channels;
    has_b = b < channels;
  }
};
template <typename T>
__device__ __forceinline__ float2 load(const T* row, const Spot& s) {
  return make_float2(s.has_a ? static_cast<float>(row[s.a]) : 0.f, s.has_b ? static_cast<float>(row[s.b]) : 0.f);
}
// a pair as it lies in memory
template <typename T>
struct RawPair {
  T a, b;
  __device__ __forceinline__ void zero() { a = b = static_cast<T>(0.f); }
  __device__ __forceinline__ void load(const T* row, const Spot& s) {  // channels that are not there stay 0
    if (s.has_a) a = row[s.a];
    if (s.has_b) b = row[s.b];
  }
  __device__ __forceinline__ float2 value() const { return make_float2(static_cast<float>(a), static_cast<float>(b)); }
};
template <typename T>
__device__ __forceinline__ void store(T* row, const Spot& s, float2 v) {
  if (s.has_a) row[s.a] = static_cast<T>(v.x);
  if (s.has_b) row[s.b] = static_cast<T>(v.y);
}
__device__ __forceinline__ float2 turned(float2 v, float2 t) { return make_float2(v.x * t.x - v.y * t.y, v.y * t.x + v.x * t.y); }
__device__ __forceinline__ float2 turned_back(float2 v, float2 t) { return make_float2(v.x * t.x + v.y * t.y, v.y * t.x - v.x * t.y); }

// Each of N (a power of two) sums over a team of `team` lanes, on all of its lanes.
template <int N>
__device__ __forceinline__ void team_sums(float (&v)[N], int team) {
  const int lane = threadIdx.x & 31;
  if (N > 1 && team >= N) {
    // lanes keep the sums whose number's bit is theirs and give the others away
#pragma unroll
    for (int o = 1; o < N; o *= 2) {
#pragma unroll
      for (int k = 0; k < N / 2 / o; ++k) {
        const bool odd = (lane & o) != 0;
        const float keep = odd ? v[2 * k + 1] : v[2 * k], give = odd ? v[2 * k] : v[2 * k + 1];
        v[k] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
      }
    }
    float sum = v[0];  // number lane % N's
    for (int o = N; o < team; o *= 2) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = __shfl_sync(0xFFFFFFFFu, sum, (lane & ~(N - 1)) | k);
  } else {
    for (int o = team >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xFFFFFFFFu, v[k], o);
    }
  }
}

// Rows of a team at a time (the next ones are loaded while these are worked on), and blocks that an SM holds. Half as
// many rows: 65536 x 16 heads x 37 forward 114 us for 111, x 100 202 for 171, x 151 289 for 260 (backward 417 for
// 370); two blocks at 37 channels 129. Without loads ahead: x 100 backward 318 for 253, x 151 482 for 370.
template <int NV>
constexpr int kForwardRows = NV == 1 ? 8 : NV <= 3 ? 4 : 2;
template <int NV>
constexpr int kBackwardRows = NV == 1 ? 4 : NV <= 3 ? 2 : 1;
template <int NV>
constexpr int kResident = NV == 1 ? 3 : NV <= 4 ? 2 : 1;

// Warps take q's items from the first on and k's from the last, so that few items spread over all of them.
struct Share {
  uint32_t first, stride;
  __device__ __forceinline__ explicit Share(int which) : stride(gridDim.x * kWarps) {
    const uint32_t warp = blockIdx.x * kWarps + threadIdx.x / 32;
    first = which == 0 ? warp : stride - 1 - warp;
  }
};

template <typename T, int NV, bool NORM>
__global__ void __launch_bounds__(kThreads, kResident<NV>)
    forward_kernel(const __grid_constant__ HeadsParams p, const __grid_constant__ AnyPlan plan) {
  constexpr int U = kForwardRows<NV>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, team = 1 << plan.shift, teams = 32 >> plan.shift, mine = lane >> plan.shift;
  const int warp_bytes = Rows<1>::bytes(plan.turns);
  Rows<1> rows(smem + warp * warp_bytes);
  const Constants constants(p, plan.table, smem + kWarps * warp_bytes);
  __syncthreads();
  const float inverse_c = 1.0f / static_cast<float>(p.channels);
  Spot spot[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) spot[n] = Spot(p.rotary, (lane & (team - 1)) + n * team, p.channels);
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const T* x = static_cast<const T*>(p.x[which].data);
    T* y = static_cast<T*>(p.out[which].data);
    RawPair<T> raw[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int n = 0; n < NV; ++n) raw[u][n].zero();
    float2 w[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) w[n] = load(constants.weight(p, which), spot[n]);
    const Share share(which);
#pragma unroll 1
    for (uint32_t id = share.first; id < plan.phase[which].items; id += share.stride) {
      rows.enter(p, plan, which, id);
      const auto fetch = [&](int base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const T* row = x + rows.offsets[0][min(base + u * teams + mine, rows.count - 1)];
#pragma unroll
          for (int n = 0; n < NV; ++n) raw[u][n].load(row, spot[n]);
        }
      };
      fetch(0);
      rows.find_turns(p.rotary, plan, constants);
#pragma unroll 1
      for (int base = 0; base < rows.count; base += U * teams) {
        float2 v[U][NV];
        float rstd[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          rstd[u] = 0.f;
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            v[u][n] = raw[u][n].value();
            rstd[u] += v[u][n].x * v[u][n].x + v[u][n].y * v[u][n].y;
          }
        }
        if (base + U * teams < rows.count) fetch(base + U * teams);
        if constexpr (NORM) team_sums(rstd, team);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = base + u * teams + mine;
          if (i >= rows.count) break;
          const float scale = NORM ? rsqrtf(rstd[u] * inverse_c + p.eps) : 1.f;
          T* row = y + rows.offsets[1][i];
          const float2* turns = rows.turns + rows.tables[i];
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            const Spot& s = spot[n];
            float2 m = v[u][n];
            if constexpr (NORM) m = make_float2(m.x * scale * w[n].x, m.y * scale * w[n].y);
            store(row, s, s.turned ? turned(m, turns[s.pair]) : m);
          }
        }
      }
    }
  }
}

// g = dy turned back, w = g weight, xh = x rstd: dx = rstd (w - xh mean(w xh)); a block's sums of g xh to its rows
// of the partial sums.
template <typename T, int NV>
__global__ void __launch_bounds__(kThreads, kResident<NV>)
    backward_kernel(const __grid_constant__ HeadsParams p, const __grid_constant__ AnyPlan plan, float* partial) {
  constexpr int U = kBackwardRows<NV>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, team = 1 << plan.shift, teams = 32 >> plan.shift, mine = lane >> plan.shift;
  const int warp_bytes = Rows<2>::bytes(plan.turns);
  Rows<2> rows(smem + warp * warp_bytes);
  const Constants constants(p, plan.table, smem + kWarps * warp_bytes);
  float* sums_of = reinterpret_cast<float*>(smem + kWarps * warp_bytes + Constants::bytes(plan.table, p.channels));
  __syncthreads();
  const float inverse_c = 1.0f / static_cast<float>(p.channels);
  Spot spot[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) spot[n] = Spot(p.rotary, (lane & (team - 1)) + n * team, p.channels);
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const T *x = static_cast<const T*>(p.x[which].data), *dy = static_cast<const T*>(p.dy[which].data);
    T* dx = static_cast<T*>(p.out[which].data);
    RawPair<T> raw[U][NV], raw_g[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        raw[u][n].zero();
        raw_g[u][n].zero();
      }
    float2 w[NV], dw[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      w[n] = load(constants.weight(p, which), spot[n]);
      dw[n] = make_float2(0.f, 0.f);
    }
    const Share share(which);
#pragma unroll 1
    for (uint32_t id = share.first; id < plan.phase[which].items; id += share.stride) {
      rows.enter(p, plan, which, id);
      const auto fetch = [&](int base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = min(base + u * teams + mine, rows.count - 1);
          const T *row = x + rows.offsets[0][i], *gradient = dy + rows.offsets[1][i];
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            raw[u][n].load(row, spot[n]);
            raw_g[u][n].load(gradient, spot[n]);
          }
        }
      };
      fetch(0);
      rows.find_turns(p.rotary, plan, constants);
#pragma unroll 1
      for (int base = 0; base < rows.count; base += U * teams) {
        float2 v[U][NV], g[U][NV];
        float sums[2 * U];  // squares, then w xh / rstd
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            v[u][n] = raw[u][n].value();
            g[u][n] = raw_g[u][n].value();
          }
        if (base + U * teams < rows.count) fetch(base + U * teams);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float2* turns = rows.turns + rows.tables[min(base + u * teams + mine, rows.count - 1)];
          sums[u] = sums[U + u] = 0.f;
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            const Spot& s = spot[n];
            if (s.turned) g[u][n] = turned_back(g[u][n], turns[s.pair]);
            sums[u] += v[u][n].x * v[u][n].x + v[u][n].y * v[u][n].y;
            sums[U + u] += v[u][n].x * g[u][n].x * w[n].x + v[u][n].y * g[u][n].y * w[n].y;
          }
        }
        team_sums(sums, team);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = base + u * teams + mine;
          if (i >= rows.count) break;
          const float rstd = rsqrtf(sums[u] * inverse_c + p.eps);
          const float along = -rstd * rstd * (sums[U + u] * rstd * inverse_c);  // -rstd^2 mean(w xh)
          T* row = dx + rows.offsets[2][i];
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            const float2 gr = make_float2(g[u][n].x * rstd, g[u][n].y * rstd);
            dw[n].x += gr.x * v[u][n].x;
            dw[n].y += gr.y * v[u][n].y;
            store(row, spot[n],
                  make_float2(gr.x * w[n].x + v[u][n].x * along, gr.y * w[n].y + v[u][n].y * along));
          }
        }
      }
    }
    if (partial == nullptr || p.dweight[which] == nullptr) continue;
    // the warp's teams by shuffles, then the warps through shared memory, each sum in a fixed order
    float* row = sums_of + warp * p.channels;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      for (int o = 16; o >= team; o >>= 1) {
        dw[n].x += __shfl_xor_sync(0xFFFFFFFFu, dw[n].x, o);
        dw[n].y += __shfl_xor_sync(0xFFFFFFFFu, dw[n].y, o);
      }
      if (lane < team) store(row, spot[n], dw[n]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.channels; c += kThreads) {
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) a += sums_of[k * p.channels + c];
      partial[(static_cast<int64_t>(which) * gridDim.x + blockIdx.x) * p.channels + c] = a;
    }
    __syncthreads();
  }
  let_next_kernel_start();
}

// ------------------------------------------------------------------ launches
AnyPlan plan_of(const HeadsParams& p, int lanes, int at_once, int resident) {
  AnyPlan plan{{{0, Divisor(1), Divisor(1), 1, 1}, {0, Divisor(1), Divisor(1), 1, 1}},
               Divisor(static_cast<uint32_t>(p.tokens)), Divisor(static_cast<uint32_t>(p.rotary.pairs > 0 ? p.rotary.pairs : 1)),
               static_cast<uint32_t>(static_cast<int64_t>(p.batch) * p.tokens), 0, 0, (p.rotary.pairs + 3) / 4 * 4, true};
  while ((1 << plan.shift) < lanes) ++plan.shift;
  const int step = at_once * (32 >> plan.shift), phases = p.heads[0] > 0 && p.heads[1] > 0 ? 2 : 1;
  int most_tokens = 1;
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0) continue;
    int chunks = (p.heads[i] + kRows - 1) / kRows, heads = (p.heads[i] + chunks - 1) / chunks, tokens = 1;
    if (chunks == 1) {
      tokens = kRows / heads;
      if (p.rotary.pairs > 0 && tokens * p.rotary.pairs > kItemPairs) tokens = kItemPairs / p.rotary.pairs;
      if (tokens < 1) tokens = 1;
    }
    // Fewer tokens an item, then fewer heads, where that saves time: rounds of items by their batches and half a batch for
    // what an item costs besides. In two rounds also at 3% more, since shorter items spread better: 2100 tokens of
    // 30 heads x 248 bf16 backward 41 us for 53. 3584 of 8 x 32, 30 channels turned: four tokens an item 6.9 us, two
    // 8.8, one 9.4; 8000 of 16 x 37 backward: four 33.3, two 30.8.
    const int64_t total = plan.total, warps = 148 * kWarps * resident / phases;
    const auto rounds = [&](int of_tokens, int of_heads) {
      const int64_t items = (total + of_tokens - 1) / of_tokens * ((p.heads[i] + of_heads - 1) / of_heads);
      return (items + warps - 1) / warps;
    };
    const auto cost = [&](int of_tokens, int of_heads) {  // in half batches
      return rounds(of_tokens, of_heads) * (2 * ((of_tokens * of_heads + step - 1) / step) + 1);
    };
    int64_t least = cost(tokens, heads);
    for (int t = tokens, h = heads; t > 1 || h > step;) {
      if (t > 1)
        t /= 2;
      else
        h = (h + 1) / 2 > step ? (h + 1) / 2 : step;
      const int64_t now = cost(t, h);
      if (now * (rounds(t, h) <= 2 ? 31 : 32) >= least * 32) continue;
      least = now;
      tokens = t;
      heads = h;
    }
    chunks = (p.heads[i] + heads - 1) / heads;
    if ((total + tokens - 1) / tokens * chunks >= int64_t(1) << 31) plan.fits = false;
    plan.phase[i] = {static_cast<uint32_t>((total + tokens - 1) / tokens * chunks), Divisor(static_cast<uint32_t>(chunks)),
                     Divisor(static_cast<uint32_t>(heads)), tokens, heads};
    if (tokens > most_tokens) most_tokens = tokens;
  }
  plan.turns = (most_tokens * p.rotary.pairs + 3) / 4 * 4;
  return plan;
}

int blocks_of(const AnyPlan& plan, int resident) {
  const int64_t want = (static_cast<int64_t>(plan.phase[0].items) + plan.phase[1].items + kWarps - 1) / kWarps, most = 148 * resident;
  return static_cast<int>(want < most ? want : most);
}

// Calls f(NV as an integral constant, lanes a team at least)
template <typename F>
int dispatch(int channels, F&& f) {
  const int pairs = (channels + 1) / 2;
  if (pairs <= 32) return f(std::integral_constant<int, 1>{}, pairs);
  if (pairs <= 64) return f(std::integral_constant<int, 2>{}, 32);
  if (pairs <= 96) return f(std::integral_constant<int, 3>{}, 32);
  if (pairs <= 128) return f(std::integral_constant<int, 4>{}, 32);
  if (pairs <= 192) return f(std::integral_constant<int, 6>{}, 32);
  return f(std::integral_constant<int, 8>{}, 32);
}

template <typename K>
int allow_shared(K kernel, size_t bytes) {
  if (bytes <= 48 * 1024) return 0;
  return static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
}

}  // namespace

template <typename T>
int forward_any(const HeadsParams& p, cudaStream_t stream) {
  return dispatch(p.channels, [&](auto nv, int lanes) {
    constexpr int NV = decltype(nv)::value;
    const AnyPlan plan = plan_of(p, lanes, kForwardRows<NV>, kResident<NV>);
    if (!plan.fits) return static_cast<int>(cudaErrorInvalidValue);
    const size_t smem = kWarps * Rows<1>::bytes(plan.turns) + Constants::bytes(plan.table, p.channels);
    auto kernel = p.norm ? forward_kernel<T, NV, true> : forward_kernel<T, NV, false>;
    const int rc = allow_shared(kernel, smem);
    if (rc != 0) return rc;
    kernel<<<blocks_of(plan, kResident<NV>), kThreads, smem, stream>>>(p, plan);
    return static_cast<int>(cudaGetLastError());
  });
}

template <typename T>
int backward_any(const HeadsParams& p, float* part, cudaStream_t stream) {
  const bool sums = p.dweight[0] != nullptr || p.dweight[1] != nullptr;
  return dispatch(p.channels, [&](auto nv, int lanes) {
    constexpr int NV = decltype(nv)::value;
    const AnyPlan plan = plan_of(p, lanes, kBackwardRows<NV>, kResident<NV>);
    if (!plan.fits) return static_cast<int>(cudaErrorInvalidValue);
    const size_t smem = kWarps * Rows<2>::bytes(plan.turns) + Constants::bytes(plan.table, p.channels) +
                        sizeof(float) * kWarps * Constants::padded(p.channels);
    const int rc = allow_shared(backward_kernel<T, NV>, smem);
    if (rc != 0) return rc;
    const int blocks = blocks_of(plan, kResident<NV>);
    backward_kernel<T, NV><<<blocks, kThreads, smem, stream>>>(p, plan, sums ? part : nullptr);
    const int launched = static_cast<int>(cudaGetLastError());
    return launched != 0 || !sums ? launched : reduce(part, p, blocks, stream);
  });
}

template int forward_any<float>(const HeadsParams&, cudaStream_t);
template int forward_any<__nv_bfloat16>(const HeadsParams&, cudaStream_t);
template int backward_any<float>(const HeadsParams&, float*, cudaStream_t);
template int backward_any<__nv_bfloat16>(const HeadsParams&, float*, cudaStream_t);

}  // namespace heads
}  // namespace ffb
