// Queries and keys of each head before an attention: divided by their root mean square, scaled by a weight,
// turned in pairs by their positions' angles, and the backward pass; the rotation alone as well.
//
// A warp takes a token's heads, a team of lanes a head: a lane holds the same pairs of channels of every
// head that comes to its team. So the warp finds the token's cosines and sines once for all heads (into
// shared memory, each pair by one lane). In the backward pass a lane also adds up the weight's gradient of its
// channels over all heads and tokens that it meets.
//
// Heads come through a ring in shared memory that belongs to the lane alone: each lane copies its own 16 bytes
// asynchronously a few steps (and tokens) ahead, and needs no barrier to read them. What is in flight then does
// not depend on registers.
//
// Heads that are not whole runs of 8 or 16 bytes a lane take heads_any.cu.
//
// Measured on one B200 (device time, inputs past L2; a plain copy moves 6.55 TB/s; boxes differ by 5%):
//   65536 tokens, 32 + 8 heads x 128 bf16          forward 214 us (6.3 TB/s), backward 339 (5.9)
//   2 x 24960 tokens, 24 + 24 heads x 128 bf16     rotation alone 207 us (5.9 TB/s)
//   65536 tokens, 16 + 16 heads x 48 bf16          forward 86 us (4.7 TB/s), backward 141 (4.3)
//   65536 tokens, 16 + 16 heads x 24 bf16          forward 67 us (3.0 TB/s), backward 109 (2.8)
//   500000 tokens, 4 + 4 heads x 32 bf16           forward 131 us (3.9 TB/s), backward 192 (4.0)
// In the first case 16 warps an SM issue in 60% of the slots: 13 instructions for 32 channels forward and 21 backward.
// A token costs a crew about as much as two to four steps of its heads (angles, addresses, the weight's values), so
// crews of a warp share it where the issue is the limit (plan_of).
// Before the ring, with heads loaded straight to registers: forward 247 us, backward 670 (or 461 with half the
// channels a lane). Without effect or slower: three blocks an SM, more slots, a table of negative sines, two heads of a
// team at a time, q and k in blocks of their own (a token's angles are then found twice: forward 264 us).
#include <string.h>

#include <type_traits>

#include "heads.cuh"
#include "launch.cuh"
#include "mx8.cuh"

namespace ffb {
namespace heads {
namespace {

// A token's position on axis `axis` (0 past the last axis).
__device__ __forceinline__ double place_of(const RotaryParams& r, uint32_t b, uint32_t t, int axis) {
  if (r.pairs == 0 || axis >= r.axes) return 0.0;
  const int64_t i = b * r.batch + t * r.token + axis * r.axis;
  return position_at(r, i);
}

// A token's cosines and sines of `slots` pairs (those past the table's: no turn) to a crew's shared memory, from
// its places on the crew's lanes.
__device__ __forceinline__ void find_turns(const RotaryParams& r, const Constants& constants, double place, int slots, int crew_lanes,
                                           float* cosines, float* sines) {
  __syncwarp();
  const int lane = threadIdx.x & (crew_lanes - 1), before = (threadIdx.x & 31) - lane;
  for (int first = 0; first < slots; first += crew_lanes) {
    const int j = first + lane;
    const double at = __shfl_sync(0xFFFFFFFFu, place, before + (j < r.pairs ? constants.axes[j] : 0));
    if (j >= slots) continue;
    const float2 t = j < r.pairs ? turn_of(at * constants.quarters[j], r.inverse ? 0x80000000u : 0u) : make_float2(1.f, 0.f);
    cosines[j] = t.x;
    sines[j] = t.y;
  }
  __syncwarp();
}

// P elements side by side in memory
template <typename T, int P>
struct Run {
  uint32_t w[P * sizeof(T) / 4];
  __device__ __forceinline__ void load(const T* p) {  // whole 16 bytes
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w)) / 16; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      memcpy(w + 4 * i, &v, 16);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(w) == 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(w)) / 16; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
  }
  __device__ __forceinline__ void set_two(int i, float x, float y) {  // elements i (even) and i + 1
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(x);
      w[i + 1] = __float_as_uint(y);
    } else {
      w[i / 2] = pack_bf16(x, y);
    }
  }
};
// A lane's P pairs of a head: their first channels `a` and second channels `b`.
template <int P>
struct Pairs {
  Lanes<P> a, b;
};

// Where a lane's P pairs lie: runs of P channels at `a` and `b`, which are the pairs' first and second channels,
// or with INTER two runs of P / 2 neighbouring pairs (a team's runs at `a` lie side by side, and so do those at `b`,
// so that its accesses take whole sectors). The pairs' angles lie at `table_a` and with INTER the second run's at
// `table_b`.
template <int P>
struct Spot {
  int a, b;                // element offsets in a head
  int table_a, table_b;
  int turned_a, turned_b;  // how many of the pairs (with INTER of each run's) are turned: the first ones
  bool there;              // whether the lane has a run
};
__device__ __forceinline__ int clamped(int v, int most) { return v < 0 ? 0 : v < most ? v : most; }
template <int P, bool INTER>
__device__ __forceinline__ Spot<P> spot_of(const RotaryParams& r, int chunk, int channels) {
  Spot<P> s;
  if constexpr (INTER) {
    s.table_a = chunk * (P / 2);
    s.table_b = channels / 4 + s.table_a;
    s.a = chunk * P;
    s.b = channels / 2 + s.a;
    s.turned_a = clamped(r.pairs - s.table_a, P / 2);
    s.turned_b = clamped(r.pairs - s.table_b, P / 2);
    s.there = s.a < channels / 2;
  } else {
    s.table_a = s.table_b = chunk * P;
    s.turned_a = s.turned_b = clamped(r.pairs - s.table_a, P);
    s.a = s.turned_a > 0 ? s.table_a : 2 * s.table_a;
    s.b = s.turned_a > 0 ? r.pairs + s.table_a : s.a + P;
    s.there = chunk * 2 * P < channels;
  }
  return s;
}

template <typename T, int P>
struct RawPairs {
  Run<T, P> a, b;
  __device__ __forceinline__ void store(T* head, const Spot<P>& s) const {
    if (!s.there) return;
    a.store(head + s.a);
    b.store(head + s.b);
  }
};
template <typename T, int P, bool INTER>
__device__ __forceinline__ Pairs<P> widen(const RawPairs<T, P>& raw) {
  Pairs<P> v;
#pragma unroll
  for (int i = 0; i < P; i += 2) {
    if constexpr (INTER) {
      const Run<T, P>& run = i < P / 2 ? raw.a : raw.b;
      const int e = 2 * i - (i < P / 2 ? 0 : P);
      v.a.p[i / 2] = f32x2(run.get(e), run.get(e + 2));
      v.b.p[i / 2] = f32x2(run.get(e + 1), run.get(e + 3));
    } else {
      v.a.p[i / 2] = f32x2(raw.a.get(i), raw.a.get(i + 1));
      v.b.p[i / 2] = f32x2(raw.b.get(i), raw.b.get(i + 1));
    }
  }
  return v;
}
template <typename T, int P, bool INTER>
__device__ __forceinline__ RawPairs<T, P> narrow(const Pairs<P>& v) {
  RawPairs<T, P> raw;
#pragma unroll
  for (int i = 0; i < P; i += 2) {
    if constexpr (INTER) {
      Run<T, P>& run = i < P / 2 ? raw.a : raw.b;
      const int e = 2 * i - (i < P / 2 ? 0 : P);
      run.set_two(e, v.a.get(i), v.b.get(i));
      run.set_two(e + 2, v.a.get(i + 1), v.b.get(i + 1));
    } else {
      raw.a.set_two(i, v.a.get(i), v.a.get(i + 1));
      raw.b.set_two(i, v.b.get(i), v.b.get(i + 1));
    }
  }
  return raw;
}

// a weight's values (in shared memory) at a lane's pairs
template <int P, bool INTER>
__device__ __forceinline__ Pairs<P> weight_of(const float* weight, const Spot<P>& s) {
  if (!s.there) return {Lanes<P>(0.f), Lanes<P>(0.f)};
  RawPairs<float, P> raw;
  raw.a.load(weight + s.a);
  raw.b.load(weight + s.b);
  return widen<float, P, INTER>(raw);
}

// a table's values for a lane's pairs
template <int P, bool INTER>
__device__ __forceinline__ Lanes<P> from_table(const float* table, const Spot<P>& s) {
  Lanes<P> v;
  if constexpr (P == 4 && INTER) {
    const float2 x = *reinterpret_cast<const float2*>(table + s.table_a), y = *reinterpret_cast<const float2*>(table + s.table_b);
    v.p[0] = f32x2(x.x, x.y);
    v.p[1] = f32x2(y.x, y.y);
  } else {
#pragma unroll
    for (int i = 0; i < P / 4; ++i) {
      const float* from = INTER && i >= P / 8 ? table + s.table_b + 4 * (i - P / 8) : table + s.table_a + 4 * i;
      const float4 t = *reinterpret_cast<const float4*>(from);
      v.p[2 * i] = f32x2(t.x, t.y);
      v.p[2 * i + 1] = f32x2(t.z, t.w);
    }
  }
  return v;
}
template <int P>
__device__ __forceinline__ Lanes<P> negative(const Lanes<P>& v) {
  return v.each([](float f) { return -f; });
}
// the turned pairs of y, the others of x: what is not turned never meets another channel's value
template <int P, bool INTER>
__device__ __forceinline__ void keep_unturned(Pairs<P>& y, const Pairs<P>& x, const Spot<P>& s) {
  if (s.turned_a + (INTER ? s.turned_b : 0) == P) return;
  const auto turned = [&](int i) { return INTER && i >= P / 2 ? i - P / 2 < s.turned_b : i < s.turned_a; };
#pragma unroll
  for (int i = 0; i < P; i += 2) {
    y.a.p[i / 2] = f32x2(turned(i) ? y.a.get(i) : x.a.get(i), turned(i + 1) ? y.a.get(i + 1) : x.a.get(i + 1));
    y.b.p[i / 2] = f32x2(turned(i) ? y.b.get(i) : x.b.get(i), turned(i + 1) ? y.b.get(i + 1) : x.b.get(i + 1));
  }
}

// the sums over a team of `team` lanes, a power of two
template <int N>
__device__ __forceinline__ void team_sums(float (&v)[N], int team) {
#pragma unroll 1
  for (int o = team >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
  }
}

// How a launch shares its work: an item is a token's next `per` heads, and a crew of 2^crew lanes takes it in teams
// of 2^shift lanes (a warp is one crew, or several where a token's heads do not fill it: its crews then take one
// item each, all of the same steps). `slots` pairs in a crew's table.
struct Plan {
  uint32_t items;
  Divisor chunks, tokens;
  int per, shift, crew, slots;
};
// A lane's place in its warp.
struct Lane {
  int lane, team, teams, mine;  // lanes a team, teams a crew, this one's team in its crew
  int to_teams;                 // log2 of teams
  uint32_t crew, crews;         // this one's crew in the warp, crews a warp
  __device__ __forceinline__ explicit Lane(const Plan& plan)
      : lane(threadIdx.x & 31), team(1 << plan.shift), teams(1 << (plan.crew - plan.shift)),
        mine((lane & ((1 << plan.crew) - 1)) >> plan.shift), to_teams(plan.crew - plan.shift),
        crew(static_cast<uint32_t>(lane) >> plan.crew), crews(32u >> plan.crew) {}
  __device__ __forceinline__ int teams_heads(int count) const { return (count - mine + teams - 1) >> to_teams; }  // of `count` heads
  __device__ __forceinline__ int steps(int count) const { return (count + teams - 1) >> to_teams; }
};

// ---- a lane's ring of S slots for NT tensors
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// A crew's item: a token's heads `first` to `last` of q's and then k's, a phase each. Past the last item nothing is
// there, but phases and steps are an item's.
struct Place {
  uint32_t b, t;
  int first, last;
  bool there;
  __device__ __forceinline__ Place(const Plan& plan, uint32_t id) : there(id < plan.items) {
    if (!there) id = 0;
    const uint32_t token = plan.chunks.quotient(id);
    b = plan.tokens.quotient(token);
    t = token - b * plan.tokens.d;
    first = (id - token * plan.chunks.d) * plan.per;
    last = first + plan.per;
  }
  __device__ __forceinline__ int begin(const HeadsParams& p, int which) const { return max(first - (which == 0 ? 0 : p.heads[0]), 0); }
  __device__ __forceinline__ int end(const HeadsParams& p, int which) const {
    return min(last - (which == 0 ? 0 : p.heads[0]), p.heads[which]);
  }
};

template <int BYTES>
__device__ __forceinline__ void read_shared(uint32_t* w, uint32_t from) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(from) : "memory");
  else
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(from) : "memory");
}

// A warp's loads of the steps of its items, a head of every team a step: through the ring, S steps ahead, each lane's own
// 16 bytes by itself.
template <typename T, int P, int NT, int S>
struct Stream {
  static constexpr int kPiece = P * sizeof(T) >= 16 ? 16 : 8;                  // bytes of a copy
  static constexpr int kPieces = P * static_cast<int>(sizeof(T)) / kPiece;     // of a run
  static constexpr int kRow = kPiece * kThreads;                               // bytes of a piece of all threads
  static constexpr int kSlot = NT * 2 * kPieces * kRow, kBytes = S * kSlot;    // bytes of a slot and of the ring

  const HeadsParams& p;
  const Plan& plan;
  const Spot<P>& spot;
  const Lane& my;
  uint32_t id, slot, last_slot;  // the warp's first item; addresses of this lane's piece
  int which, left, steps;
  Place place;
  int64_t step[NT];  // elements from one of the team's heads to the next
  const T* at[NT];

  __device__ __forceinline__ Stream(const HeadsParams& params, const Plan& plan_of, const Spot<P>& spot_of, const Lane& lane, uint32_t first,
                                    uint8_t* smem)
      : p(params), plan(plan_of), spot(spot_of), my(lane), id(first), which(-1), left(0), place(plan_of, first + lane.crew) {
    slot = smem_u32(smem) + threadIdx.x * kPiece;
    last_slot = slot + (S - 1) * kSlot;
    enter();
#pragma unroll 1
    for (int k = 0; k < S; ++k) fetch();
  }

  // to the next phase that has heads, of this item or the next
  __device__ __forceinline__ void enter() {
    while (id < plan.items) {
      if (++which == 2) {
        id += gridDim.x * kWarps * my.crews;
        which = -1;
        if (id < plan.items) place = Place(plan, id + my.crew);
        continue;
      }
      const int begin = place.begin(p, which), count = place.end(p, which) - begin;
      if (count <= 0) continue;
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        const HeadView& v = k == 0 ? p.x[which] : p.dy[which];
        at[k] = static_cast<const T*>(v.data) + (place.b * v.batch + place.t * v.token + (begin + my.mine) * v.head);
        step[k] = my.teams * v.head;
      }
      left = place.there ? my.teams_heads(count) : 0;
      steps = my.steps(count);
      return;
    }
  }

  // starts the loads of the next step
  __device__ __forceinline__ void fetch() {
    if (id < plan.items) {
      if (left > 0 && spot.there) {
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int c = 0; c < kPieces; ++c) {
            const uint32_t to = slot + (k * 2 * kPieces + c) * kRow;
            copy_async<kPiece>(to, at[k] + spot.a + c * kPiece / sizeof(T));
            copy_async<kPiece>(to + kPieces * kRow, at[k] + spot.b + c * kPiece / sizeof(T));
          }
      }
      --left;
#pragma unroll
      for (int k = 0; k < NT; ++k) at[k] += step[k];
      if (--steps == 0) enter();
    }
    commit_copies();
    slot = slot == last_slot ? last_slot - (S - 1) * kSlot : slot + kSlot;
  }

  // The oldest step's values; then its slot is free (nobody else reads it). The caller fetches the next after it
  // has widened them. What comes for channels and heads that are not there means nothing.
  __device__ __forceinline__ void take(RawPairs<T, P> (&raw)[NT]) {
    wait_copies<S - 1>();
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        const uint32_t from = slot + (k * 2 * kPieces + c) * kRow;
        read_shared<kPiece>(raw[k].a.w + c * (kPiece / 4), from);
        read_shared<kPiece>(raw[k].b.w + c * (kPiece / 4), from + kPieces * kRow);
      }
  }
};

// Slots of the rings, and blocks that an SM holds. 65536 tokens of 40 heads x 128 in bf16: forward 214 us with two blocks
// (111 registers a thread) and 3, 4 or 6 slots, 260 with three (80 registers, 150 bytes of them spilled). Backward,
// compared when a warp took a token (plan_of's crews now take 339 to 355 us): 371 us with 3 slots, 384 with 6, 398 with
// one block, 624 with three. At two blocks the bf16 backward kernels' 128 registers spill 14 to 62 bytes.
constexpr int kForwardSlots = 3, kBackwardSlots = 3;
template <typename T, int P>
constexpr int kResident = P * static_cast<int>(sizeof(T)) > 16 ? 1 : 2;

// Forward. NORM: the norm and its weight. ALL: every pair is turned.
template <typename T, int P, bool INTER, bool ALL, bool NORM>
__global__ void __launch_bounds__(kThreads, kResident<T, P>)
    heads_kernel(const __grid_constant__ HeadsParams p, const __grid_constant__ Plan plan) {
  using Heads = Stream<T, P, 1, kForwardSlots>;
  extern __shared__ __align__(16) uint8_t smem[];
  const Lane my(plan);
  const int warp = threadIdx.x / 32, tables = kWarps * my.crews;
  const uint32_t first = (blockIdx.x * kWarps + warp) * my.crews, stride = gridDim.x * tables;  // the warp's items
  float* cosines = reinterpret_cast<float*>(smem + Heads::kBytes) + (warp * my.crews + my.crew) * 2 * plan.slots;
  float* sines = cosines + plan.slots;
  const float inverse_c = 1.0f / static_cast<float>(p.channels);
  const Spot<P> spot = spot_of<P, INTER>(p.rotary, my.lane & (my.team - 1), p.channels);
  const int crew_lanes = 1 << plan.crew, axis = my.lane & (crew_lanes - 1);
  Place after(plan, first + my.crew);
  double ahead = place_of(p.rotary, after.b, after.t, axis);  // the next item's
  Heads stream(p, plan, spot, my, first, smem);
  const Constants constants(p, plan.slots, smem + Heads::kBytes + tables * 2 * plan.slots * sizeof(float));
  __syncthreads();
#pragma unroll 1
  for (uint32_t id = first; id < plan.items; id += stride) {
    const Place place = after;
    find_turns(p.rotary, constants, ahead, plan.slots, crew_lanes, cosines, sines);
    if (id + stride < plan.items) {
      after = Place(plan, id + stride + my.crew);
      ahead = place_of(p.rotary, after.b, after.t, axis);
    }
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
      const int begin = place.begin(p, which), count = place.end(p, which) - begin;
      if (count <= 0) continue;
      const HeadView& out = p.out[which];
      T* y_head = static_cast<T*>(out.data) + (place.b * out.batch + place.t * out.token + (begin + my.mine) * out.head);
      const int64_t out_head = my.teams * out.head;
      int left = place.there ? my.teams_heads(count) : 0;
      Pairs<P> c, s;  // cosines, and sines by the other channel's weight (a's negative)
      const Lanes<P> cosine = from_table<P, INTER>(cosines, spot), sine = from_table<P, INTER>(sines, spot);
      if constexpr (NORM) {
        const Pairs<P> w = weight_of<P, INTER>(constants.weight(p, which), spot);
        c = {cosine * w.a, cosine * w.b};
        s = {negative(sine) * w.b, sine * w.a};
      } else {
        c = {cosine, cosine};
        s = {negative(sine), sine};
      }
#pragma unroll 1
      for (int step = my.steps(count); step > 0; --step) {
        RawPairs<T, P> raw[1];
        stream.take(raw);
        Pairs<P> v = widen<T, P, INTER>(raw[0]);
        stream.fetch();
        if constexpr (NORM) {
          float sum[1] = {v.a.dot(v.a) + v.b.dot(v.b)};
          if (!spot.there) sum[0] = 0.f;
          team_sums(sum, my.team);
          const Lanes<P> rstd(rsqrtf(sum[0] * inverse_c + p.eps));
          v = {v.a * rstd, v.b * rstd};
        }
        if (left > 0) {
          Pairs<P> y = {fma(v.a, c.a, v.b * s.a), fma(v.b, c.b, v.a * s.b)};
          // a cosine of 1 leaves the weight
          if constexpr (!ALL) keep_unturned<P, INTER>(y, {v.a * c.a, v.b * c.b}, spot);
          narrow<T, P, INTER>(y).store(y_head, spot);
        }
        --left;
        y_head += out_head;
      }
    }
  }
}

// Backward: g = dy turned back, w = g weight, xh = x rstd: dx = rstd (w - xh mean(w xh)). A block's sums of g xh
// over its items go to its rows of the partial sums, q's rows before k's.
template <typename T, int P, bool INTER, bool ALL>
__global__ void __launch_bounds__(kThreads, kResident<T, P>)
    heads_bwd_kernel(const __grid_constant__ HeadsParams p, const __grid_constant__ Plan plan, float* partial) {
  using Heads = Stream<T, P, 2, kBackwardSlots>;
  extern __shared__ __align__(16) uint8_t smem[];
  const Lane my(plan);
  const int warp = threadIdx.x / 32, tables = kWarps * my.crews;
  const uint32_t first = (blockIdx.x * kWarps + warp) * my.crews, stride = gridDim.x * tables;  // the warp's items
  float* cosines = reinterpret_cast<float*>(smem + Heads::kBytes) + (warp * my.crews + my.crew) * 2 * plan.slots;
  float* sines = cosines + plan.slots;
  const float inverse_c = 1.0f / static_cast<float>(p.channels);
  const Spot<P> spot = spot_of<P, INTER>(p.rotary, my.lane & (my.team - 1), p.channels);
  Pairs<P> dw[2];
  dw[0] = dw[1] = {Lanes<P>(0.f), Lanes<P>(0.f)};
  const int crew_lanes = 1 << plan.crew, axis = my.lane & (crew_lanes - 1);
  Place after(plan, first + my.crew);
  double ahead = place_of(p.rotary, after.b, after.t, axis);  // the next item's
  Heads stream(p, plan, spot, my, first, smem);
  const Constants constants(p, plan.slots, smem + Heads::kBytes + tables * 2 * plan.slots * sizeof(float));
  __syncthreads();
#pragma unroll 1
  for (uint32_t id = first; id < plan.items; id += stride) {
    const Place place = after;
    find_turns(p.rotary, constants, ahead, plan.slots, crew_lanes, cosines, sines);
    if (id + stride < plan.items) {
      after = Place(plan, id + stride + my.crew);
      ahead = place_of(p.rotary, after.b, after.t, axis);
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int begin = place.begin(p, which), count = place.end(p, which) - begin;
      if (count <= 0) continue;
      const HeadView& out = p.out[which];
      T* dx_head = static_cast<T*>(out.data) + (place.b * out.batch + place.t * out.token + (begin + my.mine) * out.head);
      const int64_t out_head = my.teams * out.head;
      int left = place.there ? my.teams_heads(count) : 0;
      const Pairs<P> w = weight_of<P, INTER>(constants.weight(p, which), spot);
#pragma unroll 1
      for (int step = my.steps(count); step > 0; --step) {
        RawPairs<T, P> raw[2];
        stream.take(raw);
        const Lanes<P> c = from_table<P, INTER>(cosines, spot), s = from_table<P, INTER>(sines, spot);
        const Pairs<P> v = widen<T, P, INTER>(raw[0]), d = widen<T, P, INTER>(raw[1]);
        Pairs<P> g = {fma(d.a, c, d.b * s), fma(d.b, c, negative(d.a * s))};
        if constexpr (!ALL) keep_unturned<P, INTER>(g, d, spot);
        float sums[2] = {v.a.dot(v.a) + v.b.dot(v.b), (v.a * w.a).dot(g.a) + (v.b * w.b).dot(g.b)};
        if (!spot.there) sums[0] = sums[1] = 0.f;
        stream.fetch();
        team_sums(sums, my.team);
        if (left > 0) {
          const float rstd = rsqrtf(sums[0] * inverse_c + p.eps);
          const Lanes<P> along(-rstd * rstd * (sums[1] * rstd * inverse_c));  // -rstd^2 mean(w xh)
          const Pairs<P> gr = {g.a * Lanes<P>(rstd), g.b * Lanes<P>(rstd)};
          dw[which] = {fma(gr.a, v.a, dw[which].a), fma(gr.b, v.b, dw[which].b)};
          const Pairs<P> y = {fma(v.a, along, gr.a * w.a), fma(v.b, along, gr.b * w.b)};
          narrow<T, P, INTER>(y).store(dx_head, spot);
        }
        --left;
        dx_head += out_head;
      }
    }
  }
  if (partial == nullptr) return;
  let_next_kernel_start();
  // the warp's teams by shuffles, then the warps through shared memory, each sum in a fixed order
  float* sums = reinterpret_cast<float*>(smem);
  float* row = sums + warp * p.channels;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (p.dweight[which] == nullptr) continue;
    __syncthreads();
    for (int o = 16; o >= my.team; o >>= 1) {
      dw[which].a = dw[which].a.each([&](float f) { return f + __shfl_xor_sync(0xFFFFFFFFu, f, o); });
      dw[which].b = dw[which].b.each([&](float f) { return f + __shfl_xor_sync(0xFFFFFFFFu, f, o); });
    }
    if (my.lane < my.team && spot.there) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int at = !INTER ? spot.a + j : j < P / 2 ? spot.a + 2 * j : spot.b + 2 * j - P;
        row[at] = dw[which].a.get(j);
        row[INTER ? at + 1 : spot.b + j] = dw[which].b.get(j);
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.channels; c += kThreads) {
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) a += sums[k * p.channels + c];
      partial[(static_cast<int64_t>(which) * gridDim.x + blockIdx.x) * p.channels + c] = a;
    }
  }
}

// a weight's gradient from the blocks' partial sums (q's rows first), in a fixed order: 32 channels a block
__global__ void __launch_bounds__(1024)
    heads_reduce_kernel(const float* __restrict__ part, float* dq_weight, float* dk_weight, int blocks, int channels) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, r = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
  float* out = blockIdx.y == 0 ? dq_weight : dk_weight;
  const float* rows = part + static_cast<int64_t>(blockIdx.y) * blocks * channels;
  wait_for_kernel_before();
  if (out == nullptr) return;
  float v = 0.f;
  if (c < channels)
    for (int i = r; i < blocks; i += 32) v += rows[static_cast<int64_t>(i) * channels + c];
  s[r][lane] = v;
  __syncthreads();
  if (r == 0 && c < channels) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) a += s[k][lane];
    out[c] = a;
  }
}

// ------------------------------------------------------------------ launches
bool on(const HeadView& v, int elements, int size, const HeadsParams& p, int heads) {
  return (reinterpret_cast<uintptr_t>(v.data) % static_cast<uintptr_t>(elements * size < 16 ? elements * size : 16)) == 0 &&
         (p.batch <= 1 || v.batch % elements == 0) && (p.tokens <= 1 || v.token % elements == 0) && (heads <= 1 || v.head % elements == 0);
}

// whether runs of P channels are whole and aligned in every tensor of the call
bool runs_of(const HeadsParams& p, int P, int size, bool backward) {
  const RotaryParams& r = p.rotary;
  if (p.channels % (2 * P) != 0 || p.channels / (2 * P) > 32) return false;
  if (!r.interleaved && r.pairs % P != 0) return false;
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0) continue;
    if (!on(p.x[i], P, size, p, p.heads[i]) || !on(p.out[i], P, size, p, p.heads[i])) return false;
    if (backward && !on(p.dy[i], P, size, p, p.heads[i])) return false;
  }
  return true;
}

constexpr int kNoRuns = -1;

// Calls f(P, INTER, ALL as integral constants, lanes a team at least): runs of 16 bytes where they are whole and aligned
// (fp32 heads of more than 256 channels in two of them), else of half that, else kNoRuns.
template <typename T, typename F>
int dispatch_heads(const HeadsParams& p, bool backward, F&& f) {
  const int size = sizeof(T);
  const auto runs = [&](auto P) {
    const int lanes = p.channels / (2 * decltype(P)::value);
    const std::true_type yes;
    const std::false_type no;
    if (2 * p.rotary.pairs == p.channels) return p.rotary.interleaved ? f(P, yes, yes, lanes) : f(P, no, yes, lanes);
    return p.rotary.interleaved ? f(P, yes, no, lanes) : f(P, no, no, lanes);
  };
  if (sizeof(T) == 4 && runs_of(p, 4, size, backward)) return runs(std::integral_constant<int, 4>{});
  if (runs_of(p, 8, size, backward)) return runs(std::integral_constant<int, 8>{});
  if (sizeof(T) == 2 && runs_of(p, 4, size, backward)) return runs(std::integral_constant<int, 4>{});
  return kNoRuns;
}

// How tokens' heads are cut into items. An item's issue time, in fortieths of a step of runs of 8: fixed work
// (addresses, the weight's values) of about two steps, a quarter of one for each round of the crew's lanes over the
// pairs' angles, and its steps; its memory time, the bytes of its heads, where the issue of a full step of 1 KB an
// input takes 40 and its memory 57 (44 of a backward step, which issues more for its three KB; fp32 a quarter more). The GPU's crews take
// the items in rounds. Smaller crews share the fixed work among more tokens of a warp and take more steps, which
// helps where the issue is the limit (65536 tokens of 16 heads x 24: 68 -> 39 us forward, 84 -> 62 backward; of 32 x 24
// 86 -> 67 and 114 -> 109; of 32 x 48 104 -> 86 and 174 -> 141) and not where the memory is (40 x 128: 214 -> 218
// forward). Where there are few tokens, a whole warp takes a token, or a part of its heads.
Plan plan_of(const HeadsParams& p, int lanes, int run, int resident, int size, bool backward) {
  const int heads = p.heads[0] + p.heads[1];
  Plan best{0, Divisor(1), Divisor(static_cast<uint32_t>(p.tokens)), heads, 0, 0, 0};
  while ((1 << best.shift) < lanes) ++best.shift;
  best.slots = run << best.shift;
  const int64_t tokens = static_cast<int64_t>(p.batch) * p.tokens, warps = 148 * kWarps * static_cast<int64_t>(resident);
  int64_t least = 0;
  const auto consider = [&](int crew, int per, int64_t chunks, int64_t steps) {
    const int64_t items = tokens * chunks, crews = warps * (32 >> crew), full = 16 * items / crews;
    const int64_t rounds = full < 16 ? 16 : full + 8;  // sixteenths; the last one is half a round in the mean
    const int64_t issue = 80 + 10 * ((best.slots + (1 << crew) - 1) >> crew) + (run == 4 ? 25 : 40) * steps;
    const int64_t memory = (backward ? 44 : 57) * static_cast<int64_t>(per) * p.channels * (size == 4 ? 5 : 2) / 1024 * (32 >> crew);
    const int64_t cost = rounds * (issue > memory ? issue : memory);
    if (least != 0 && cost >= least) return;
    least = cost;
    best.crew = crew;
    best.per = per;
    best.chunks = Divisor(static_cast<uint32_t>(chunks));
    best.items = static_cast<uint32_t>(items);
  };
  for (int crew = 5; crew >= best.shift; --crew) {
    if (p.rotary.pairs > 0 && 1 << crew < p.rotary.axes) break;
    const int step = 1 << (crew - best.shift);
    consider(crew, heads, 1, (p.heads[0] + step - 1) / step + (p.heads[1] + step - 1) / step);
    if (crew < 5) continue;  // crews of one warp take the same steps
    for (int of = (heads + step - 1) / step / 2; of >= 1 && tokens < warps; of /= 2) {  // steps an item
      consider(crew, of * step, (heads + of * step - 1) / (of * step), of);
      if (of == 1) break;
    }
  }
  return best;
}
size_t table_bytes(const Plan& plan, int channels) {
  return sizeof(float) * kWarps * (32 >> plan.crew) * 2 * plan.slots + Constants::bytes(plan.slots, channels);
}

int blocks_of(const Plan& plan, int resident) {
  const int64_t warp_items = kWarps * (32 >> plan.crew), want = (plan.items + warp_items - 1) / warp_items, most = 148 * resident;
  return static_cast<int>(want < most ? want : most);
}

template <typename T>
int forward(const HeadsParams& p, cudaStream_t stream) {
  const int rc = dispatch_heads<T>(p, false, [&](auto run, auto inter, auto all, int lanes) {
    constexpr int P = decltype(run)::value;
    constexpr bool INTER = decltype(inter)::value, ALL = decltype(all)::value;
    const Plan plan = plan_of(p, lanes, P, kResident<T, P>, sizeof(T), false);
    const size_t smem = Stream<T, P, 1, kForwardSlots>::kBytes + table_bytes(plan, p.channels);
    auto kernel = p.norm ? heads_kernel<T, P, INTER, ALL, true> : heads_kernel<T, P, INTER, ALL, false>;
    if (smem > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (e != cudaSuccess) return static_cast<int>(e);
    }
    kernel<<<blocks_of(plan, kResident<T, P>), kThreads, smem, stream>>>(p, plan);
    return static_cast<int>(cudaGetLastError());
  });
  return rc == kNoRuns ? forward_any<T>(p, stream) : rc;
}

template <typename T>
int backward(const HeadsParams& p, float* part, cudaStream_t stream) {
  const bool sums = p.dweight[0] != nullptr || p.dweight[1] != nullptr;
  const int rc = dispatch_heads<T>(p, true, [&](auto run, auto inter, auto all, int lanes) {
    constexpr int P = decltype(run)::value;
    constexpr bool INTER = decltype(inter)::value, ALL = decltype(all)::value;
    const Plan plan = plan_of(p, lanes, P, kResident<T, P>, sizeof(T), true);
    size_t smem = Stream<T, P, 2, kBackwardSlots>::kBytes + table_bytes(plan, p.channels);
    if (smem < sizeof(float) * kWarps * p.channels) smem = sizeof(float) * kWarps * p.channels;
    auto kernel = heads_bwd_kernel<T, P, INTER, ALL>;
    if (smem > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (e != cudaSuccess) return static_cast<int>(e);
    }
    const int blocks = blocks_of(plan, kResident<T, P>);
    kernel<<<blocks, kThreads, smem, stream>>>(p, plan, sums ? part : nullptr);
    const int launched = static_cast<int>(cudaGetLastError());
    return launched != 0 || !sums ? launched : reduce(part, p, blocks, stream);
  });
  return rc == kNoRuns ? backward_any<T>(p, part, stream) : rc;
}

}  // namespace

int reduce(const float* part, const HeadsParams& p, int blocks, cudaStream_t stream) {
  return launch_after(heads_reduce_kernel, dim3((p.channels + 31) / 32, 2), 1024, 0, stream, part, p.dweight[0], p.dweight[1], blocks,
                      p.channels);
}

}  // namespace heads

size_t heads_bwd_workspace_bytes(int64_t, int, int, int channels, int) {
  return static_cast<size_t>(2 * heads::kMostBlocks) * channels * sizeof(float);
}
int launch_heads(const HeadsParams& p, int is_f32, cudaStream_t stream) {
  return is_f32 ? heads::forward<float>(p, stream) : heads::forward<__nv_bfloat16>(p, stream);
}
int launch_heads_bwd(const HeadsParams& p, void* workspace, int is_f32, cudaStream_t stream) {
  float* part = static_cast<float*>(workspace);
  return is_f32 ? heads::backward<float>(p, part, stream) : heads::backward<__nv_bfloat16>(p, part, stream);
}

}  // namespace ffb
