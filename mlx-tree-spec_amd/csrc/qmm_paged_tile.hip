// Paged attention of more than 16 query rows to a key head, tree verify and prompt rows, and of all rows of bf16 heads of 192 and
// more (qmm_paged.h has the products and the softmax). Each byte of the cache serves up to 128 query rows of a workgroup: bound by
// HBM up to some 64 rows (one row of 6 heads over 200000 tokens, 4 key heads of 256: 137 us, 6.0 TB/s), past that by the matrix
// instructions and the softmax's vector instructions (64 nodes of 4 heads over 32000 tokens, 8 key heads of 128: 51.6 us, 650 TFLOP/s;
// 1000 rows over 8000: 168 us, 830 TFLOP/s).
//
// A workgroup takes up to kPagedRows query rows of one key head over one split: 8 waves with 16 QT rows each, or with two SIDES
// 4 of them on the even steps and the others with the same rows on the odd ones. The steps' keys and values go from memory to
// a ring of stages in LDS without registers (1 KB an instruction), two stages ahead, in the order in which the waves read
// them: a fragment is then 256 neighbouring bytes for 16 lanes, without bank conflicts. One barrier a stage, in front of the
// softmax, behind an exact count of the loads that may still be on their way: the softmax covers the reads of its own values and of the
// next step's keys (1000 rows 181 -> 174 us, 4 x 16 nodes of 6 heads of 256 28.4 -> 26.6).
// 8 bits: the waves together make a stage's codes bf16 numbers, in LDS, one stage ahead and behind the products of keys; each wave
// for itself would make them all again (1000 rows over 8000 tokens, 8 heads of 128: 308 -> 208 us, 4 of 256 over 4000: 426 -> 232; 4 x 16
// nodes of 6 heads of 256 over 8000: 28.6 -> 20.2).
// (Half of the waves half a stage late, so that a SIMD's two would multiply and exponentiate in turn, measured the same; so did
// priorities, 4 waves to a workgroup and two of those to a CU, and the values' products among the next step's exponentials: with
// heads of 256 those took more registers than there are.)
#include <algorithm>
#include <type_traits>

#include "qmm4_lds.h"
#include "qmm_paged.h"

namespace qmm4 {

namespace {

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * 64;
constexpr int kIds = 1024;  // page numbers held in LDS at once

template <int D, int QT, int SIDES, bool Q8>
struct TileTraits {
  using R = PagedRows<D, QT, Q8, false>;
  static constexpr int kAcross = kWaves / SIDES;          // waves side by side along the rows
  static constexpr int kRows = kAcross * 16 * QT;
  static constexpr int kStage = SIDES * R::kStep;         // tokens
  static constexpr int kPieces = D * kStage * 2 / R::E;   // 16-byte pieces of a stage: keys, then values
  static constexpr int kChunks = kPieces / 64;            // loads of them
  static constexpr int kStageBytes = kPieces * 16 + (Q8 ? 1024 : 0);  // (scales, over and over)
  static constexpr int kChunkLoads = (kChunks / 2 + kWaves / 2 - 1) / (kWaves / 2);
  static constexpr int kLoads = kChunkLoads + (Q8 ? 1 : 0);  // a wave's loads of a stage
  // A stage that is multiplied, whose values are read while the next one's keys are, and two on their way.
  static constexpr int kStages = 4;
  // A step's keys are read while the softmax before it runs, or where registers are short piece by piece in place of values.
  static constexpr bool kEarly = R::kKC * R::kKT <= 8 && !(Q8 && QT * D >= 256);
  static constexpr int kBf16 = D * kStage * 2 / 8;  // pieces of a stage as bf16 numbers
  static constexpr size_t kRing = (size_t)kStages * kStageBytes + (Q8 ? 2 * kBf16 * 16 : 0);
  static constexpr size_t kJoin = SIDES > 1 ? (size_t)kAcross * R::kHandBytes : 0;
  static constexpr size_t kLds = (kRing > kJoin ? kRing : kJoin) + kIds * 4 + 16;
  static_assert(kLds <= 160 * 1024, "LDS");
};

// Waits until at most N of the wave's loads into LDS are on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Waits for the wave's reads out of LDS and its writes to it.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ void bare_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// WIDE: pages of a stage's tokens and more.
template <int D, int QT, int SIDES, bool Q8, bool WIDE>
__global__ __launch_bounds__(kThreads) void paged_tile_kernel(PagedParams S, int block0, int blocks) {
  using T = TileTraits<D, QT, SIDES, Q8>;
  using R = PagedRows<D, QT, Q8, false>;
  constexpr int E = R::E;
  typedef __attribute__((address_space(1))) const void* global_ptr;
  typedef __attribute__((address_space(3))) void* lds_ptr;
  extern __shared__ __attribute__((aligned(16))) char s_ring[];
  int* s_ids = reinterpret_cast<int*>(s_ring + T::kLds - kIds * 4 - 16);
  int* s_odd = s_ids + kIds;  // a value that is not finite was left out
  // The row blocks of one split and key head (a unit) follow each other on one XCD (workgroups go round the 8 of them): the later
  // ones find the cache's bytes in its L2.
  int unit = blockIdx.x / (8 * blocks) * 8 + (blockIdx.x & 7), in_unit = blockIdx.x / 8 % blocks;
  if (blocks > 2) {
    // Prompts: most of the grid, made for as many splits as there may be, ends here, before anything else. Units that are few and not
    // a multiple of 8 are shared out, so that every XCD has as many blocks (1000 rows, 47 blocks of one request, over 4 key heads of 256:
    // 182 us, 343 on 4 XCDs).
    const int units = S.plan.words[0] * S.cache.heads;
    if (blockIdx.x >= (uint32_t)((units + 7) / 8 * 8) * (blocks + 7)) return;
    if (units < 64 && units % 8 != 0) {
      const int share = min(blocks, units % 4 == 0 ? 2 : units % 2 == 0 ? 4 : 8), each = (blocks + share - 1) / share;
      const int place = blockIdx.x / (8 * each) * 8 + (blockIdx.x & 7);
      unit = place / share;
      in_unit = place % share * each + blockIdx.x / 8 % each;
      if (in_unit >= blocks) return;
    }
  }
  const int item = unit / S.cache.heads, block = block0 + in_unit;
  const PagedItem I = S.plan.items()[item < S.items ? item : 0];
  if (item >= S.plan.words[0]) return;
  R W(S, I, unit - item * S.cache.heads);
  const int row0 = block * T::kRows, rows = I.rows * S.G;
  if (row0 >= rows) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), side = wave / T::kAcross, rw = wave % T::kAcross;
  const int mine = row0 + rw * 16 * QT;
  const bool active = mine < rows;
  W.load_rows(mine);

  // (Waited for here: the barriers in front of a stage's reads are bare, and the first stage may set it.)
  if (threadIdx.x == 0) *s_odd = 0;
  wait_reads();
  const int begin = I.begin;
  int end = I.end;
  // (Without ancestors nothing past the block's last row is seen.)
  if (!S.ancestors) end = min(end, W.context + min((row0 + T::kRows - 1) / S.G, I.rows - 1) + 1);
  const int shift = S.cache.page_shift, page_mask = (1 << shift) - 1, lane = W.lane;
  typedef __attribute__((address_space(4))) const int32_t* constant_ptr;
  const constant_ptr constant_table = (constant_ptr)W.table;  // (nothing in this kernel writes it: scalar loads)
  const char* keys = static_cast<const char*>(S.cache.keys);
  const char* values = static_cast<const char*>(S.cache.values);

  // A step from a stage in LDS: its products with the queries ..
  f32x4 s[QT][R::kKT];
  u32x4 vf[R::kVT];  // 8 tokens of a dimension each
  f32x4 ks[Q8 ? R::kKT : 1], vs[Q8 ? R::kKT : 1];
  const auto multiply = [&](const u32x4 (&kf)[R::kKC][R::kKT]) __attribute__((always_inline)) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int tt = 0; tt < R::kKT; ++tt) s[qt][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < R::kKC; ++c) {
#pragma unroll
      for (int tt = 0; tt < R::kKT; ++tt) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[qt][tt] = paged_mma(as_bf16x8(kf[c][tt]), W.q[qt][c], s[qt][tt]);
      }
    }
  };
  // .. and what they add to the rows.
  const auto finish = [&](int t, auto&& between) __attribute__((always_inline)) {
    bf16x8 p[QT];
    W.softmax(t, s, ks, vs, p);
#pragma unroll
    for (int dt = 0; dt < R::kVT; ++dt) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) W.o[qt][dt] = paged_mma(as_bf16x8(vf[dt]), p[qt], W.o[qt][dt]);
      between(dt);
    }
  };

  // WIDE: one page for a stage, addresses that only the scalar unit makes.
  static_assert(kPagedUnit % T::kStage == 0, "a stage begins at a multiple of its tokens");
  const int segment = WIDE ? 1 << 30 : kIds << shift;  // tokens whose pages are known at once
  // A lane's token of a key's piece, in the order of the tiles' rows.
  const int key_token = lane % T::kStage / R::kStep * R::kStep + 8 * ((lane & 15) >> 2) + 4 * (lane / 16 % R::kKT) + (lane & 3);
  constexpr int kScaleLanes = T::kStage / 4;
  constexpr int kKeyPieces = 64 / T::kStage;  // pieces of keys in one load
  // A wave's loads: neighbouring kilobytes of the stage's keys (the lower half of the waves) or of its values (the last ones of
  // either again where they do not divide). Its lanes' places in a page, those of a token on, and of a load on.
  const int mine_chunk = wave / (kWaves / 2) * (T::kChunks / 2) +
                         min(wave % (kWaves / 2) * T::kChunkLoads, T::kChunks / 2 - T::kChunkLoads);
  const bool mine_keys = wave < kWaves / 2;
  const char* mine_base = mine_keys ? keys + ((int64_t)mine_chunk * kKeyPieces << (shift + 4))
                                    : values + (mine_chunk - T::kChunks / 2) * 1024;
  const int mine_token = mine_keys ? 16 : D * 16 / E, mine_stride = mine_keys ? kKeyPieces << (shift + 4) : 1024;
  const uint32_t mine_offset = mine_keys ? ((uint32_t)(lane / T::kStage) << (shift + 4)) + key_token * 16 : lane * 16;
  const uint32_t head_bytes = D * 16 / E << shift, page_bytes = S.cache.heads * head_bytes;  // of a page (at most 2^29)
  const char* mine_head = mine_base + (int64_t)W.h * head_bytes;
  const auto page_at = [&](int tok) { return constant_table[(uint32_t)min(tok, W.length - 1) >> shift]; };
  for (int base = begin & ~page_mask; base < end; base += segment) {
    const int from = max(begin, base), to = min(end, base > (1 << 30) - segment ? end : base + segment);
    const int stages = (to - from + T::kStage - 1) / T::kStage;
    int next_page = 0;  // (as the table has it: made valid where it is used, a stage later)
    if constexpr (WIDE) {
      next_page = from == begin ? I.page : page_at(from);
    } else {
      __syncthreads();
      for (int i = threadIdx.x; i < kIds; i += kThreads) {
        const int tok = base + (i << shift);
        s_ids[i] = tok < W.length ? W.valid_page(W.table[tok >> shift]) : 0;
      }
      __syncthreads();
    }

    // Stage `st` of the segment into its place of the ring. (Tokens past the last: others of the page, or the last group again.)
    auto load = [&](int st) __attribute__((always_inline)) {
      const int t = from + st * T::kStage;
      char* ring = s_ring + (st % T::kStages) * T::kStageBytes;
      if constexpr (WIDE) {
        const uint32_t page = W.valid_page(next_page), off = t & page_mask;
        next_page = page_at(t + T::kStage);
        const char* src = mine_head + (uint64_t)page * page_bytes + off * mine_token;
#pragma unroll
        for (int j = 0; j < T::kChunkLoads; ++j)
          __builtin_amdgcn_global_load_lds((global_ptr)(src + j * mine_stride + mine_offset),
                                           (lds_ptr)(ring + (mine_chunk + j) * 1024), 16, 0, 0);
        if constexpr (Q8) {
          // 4 tokens a lane: key scales, value scales, and both again (every lane of a load writes).
          const float* src = (lane & kScaleLanes ? S.cache.value_scales : S.cache.key_scales) +
                             (((int64_t)page * S.cache.heads + W.h) << shift) + off;
          __builtin_amdgcn_global_load_lds((global_ptr)(src + (lane & (kScaleLanes - 1)) * 4), (lds_ptr)(ring + T::kPieces * 16), 16, 0, 0);
        }
      } else {
        const auto head_of = [&](int tok) { return (int64_t)s_ids[(tok - base) >> shift] * S.cache.heads + W.h; };
        const int grp = min(W.group(t + (key_token & ~7)), base + segment - 8);
        const char* kp = keys + ((head_of(grp) * (D / E) << shift) + (grp & page_mask) + (key_token & 7)) * 16;
#pragma unroll
        for (int j = 0; j < T::kChunkLoads; ++j) {
          const int chunk = mine_chunk + j;
          const char* src;
          if (chunk < T::kChunks / 2) {
            src = kp + ((int64_t)(chunk * kKeyPieces + lane / T::kStage) << (shift + 4));
          } else {
            const int f = (chunk - T::kChunks / 2) * 64 + lane, at = f / D, d = f - at * D;
            const int tok = min(W.group(t + at * E), base + segment - E) & ~(E - 1);
            src = values + (((head_of(tok) << shift) + (tok & page_mask)) / E * D + d) * 16;
          }
          __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)(ring + chunk * 1024), 16, 0, 0);
        }
        if constexpr (Q8) {
          const int tok = min(W.group(t + (lane & (kScaleLanes - 2)) * 4), base + segment - 8) + (lane & 1) * 4;
          const float* src = (lane & kScaleLanes ? S.cache.value_scales : S.cache.key_scales) + (head_of(tok) << shift) + (tok & page_mask);
          __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)(ring + T::kPieces * 16), 16, 0, 0);
        }
      }
    };

    const auto ring_of = [&](int st) { return reinterpret_cast<u32x4*>(s_ring + (st % T::kStages) * T::kStageBytes); };
    // Its keys and values as bf16 numbers.
    const auto stage_of = [&](int st) {
      if constexpr (Q8) return reinterpret_cast<u32x4*>(s_ring + T::kStages * T::kStageBytes) + (st & 1) * T::kBf16;
      else return ring_of(st);
    };
    // (Splits begin and end at whole stages, but for the last token that is seen: past that a step has no effect.)
    const auto token_of = [&](int st) { return from + st * T::kStage + side * R::kStep; };
    // The values of a stage past the context made clean in place, by all waves (once: a branch around products of clean and other
    // values would have every sum in registers twice).
    const auto clean = [&](int st) {
      u32x4* values = ring_of(st) + T::kPieces / 2;
      for (int f = threadIdx.x; f < T::kPieces / 2; f += kThreads) {
        bool odd = false;
        values[f] = clean_values(values[f], from + st * T::kStage + f / D * 8 - W.length, &odd);
        if (odd) *s_odd = 1;
      }
    };
    // 8 bits: a stage's codes as bf16 numbers, by all waves (once, and not by each wave that multiplies them).
    const auto convert = [&](int st) __attribute__((always_inline)) {
      const u32x4* from_codes = ring_of(st);
      u32x4* to_bf16 = stage_of(st);
#pragma unroll
      for (int f0 = 0; f0 < T::kPieces; f0 += kThreads) {
        const int f = f0 + threadIdx.x;
        if (T::kPieces % kThreads != 0 && f >= T::kPieces) break;
        // (16 dimensions of a token, or 16 tokens of a dimension: two pieces, a row of tokens or of dimensions apart.)
        const int v = f - T::kPieces / 2, row = v < 0 ? T::kStage : D, at = v < 0 ? f / T::kStage : v / D, i = v < 0 ? f % T::kStage : v % D;
        u32x4* to = to_bf16 + (v < 0 ? 0 : T::kBf16 / 2) + 2 * at * row + i;
        const u32x4 x = from_codes[f];
        to[0] = __builtin_bit_cast(u32x4, codes8(x[0], x[1]));
        to[row] = __builtin_bit_cast(u32x4, codes8(x[2], x[3]));
      }
    };
    // Behind it stage `st` can be read by every wave (8 bits: and the codes of the next be converted), where all up to kOnWay behind
    // `st` are loaded or on their way.
    constexpr int kOnWay = Q8 ? 2 : 1;
    const auto arrive = [&](int st) __attribute__((always_inline)) {
      if (st + kOnWay < stages) wait_loads<T::kLoads>();
      else wait_loads<0>();
      bare_barrier();
      if (Q8 || from + (st + 1) * T::kStage <= W.context) return;
      clean(st);
      wait_reads();
      bare_barrier();
    };
    u32x4 kf[R::kKC][R::kKT];
    const auto read_key = [&](int st, int c, int tt) __attribute__((always_inline)) {
      kf[c][tt] = (stage_of(st) + W.g * T::kStage + side * R::kStep + W.r16)[c * 4 * T::kStage + tt * 16];
    };
    const auto read_keys = [&](int st) __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < R::kKC; ++c)
#pragma unroll
        for (int tt = 0; tt < R::kKT; ++tt) read_key(st, c, tt);
    };
    // The next stage, and one behind those on their way into the place of one that is done.
    const auto advance = [&](int st, auto&& then) __attribute__((always_inline)) {
      if (st + 1 >= stages) return;
      if constexpr (Q8) {
        convert(st + 1);
        wait_reads();
      }
      arrive(st + 1);
      then();
      if (st + 2 + kOnWay < stages) load(st + 2 + kOnWay);
    };
    for (int st = 0; st < 1 + kOnWay && st < stages; ++st) load(st);
    if constexpr (Q8) {
      if (stages > 2) wait_loads<2 * T::kLoads>();
      else if (stages > 1) wait_loads<T::kLoads>();
      else wait_loads<0>();
      bare_barrier();
      convert(0);
      wait_reads();
    }
    arrive(0);
    if (active) read_keys(0);
    if (1 + kOnWay < stages) load(1 + kOnWay);
    if (!active) {
#pragma unroll 1
      for (int st = 0; st < stages; ++st) advance(st, [] {});
    } else {
#pragma unroll 1
      for (int st = 0; st < stages; ++st) {
        // (The keys, and all that was read before them: behind the next barrier the place of the stage before is loaded again.)
        wait_reads();
        multiply(kf);
        __builtin_amdgcn_sched_barrier(0);
        const u32x4* vr = stage_of(st) + T::kBf16 / 2 + (side * 4 + W.g) * D + W.r16;
#pragma unroll
        for (int dt = 0; dt < R::kVT; ++dt) vf[dt] = vr[dt * 16];
        if constexpr (Q8) {
          const f32x4* scales = reinterpret_cast<const f32x4*>(ring_of(st) + T::kPieces) + side * 8 + W.g * 2;
#pragma unroll
          for (int tt = 0; tt < R::kKT; ++tt) {
            ks[tt] = scales[tt];
            vs[tt] = scales[T::kStage / 4 + tt];
          }
        }
        const int next = st + 1 < stages ? st + 1 : st;
        advance(st, [&]() __attribute__((always_inline)) {
          if constexpr (T::kEarly) read_keys(next);
        });
        if constexpr (T::kEarly) {
          finish(token_of(st), [](int) {});
        } else {
          constexpr int kEach = R::kKC * R::kKT / R::kVT;
          static_assert(kEach * R::kVT == R::kKC * R::kKT, "keys in place of values");
          finish(token_of(st), [&](int dt) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) read_key(next, (dt * kEach + i) / R::kKT, (dt * kEach + i) % R::kKT);
            __builtin_amdgcn_sched_barrier(0);
          });
        }
      }
    }
    // (Every load has been waited for: the ring is free behind the next barrier.)
    __syncthreads();
    W.odd = *s_odd != 0;
    // (A whole stage was made clean, both sides' steps of it.)
    if (active) W.add_odd_values(from + side * R::kStep, to, T::kStage, T::kStage - side * R::kStep, mine);
  }

  W.sum_lanes();
  if constexpr (SIDES > 1) {
    __syncthreads();
    if (side == 1) W.hand_over(s_ring + rw * R::kHandBytes);
    __syncthreads();
    if (side == 0) W.take_over(s_ring + rw * R::kHandBytes);
  }
  if (side == 0 && active) W.write(mine);
}

template <int D, int QT, int SIDES, bool Q8, bool WIDE>
hipError_t launch_pages(const PagedParams& p, hipStream_t stream) {
  using T = TileTraits<D, QT, SIDES, Q8>;
  static LdsAllowance allowance;
  if (hipError_t e = allowance.allow(reinterpret_cast<const void*>(&paged_tile_kernel<D, QT, SIDES, Q8, WIDE>), T::kLds)) return e;
  // (At least 128: units that are shared out, fewer than 64, take up to twice as many places.)
  const int64_t units = std::max<int64_t>(128, ((int64_t)p.items * p.cache.heads + 7) / 8 * 8);
  const int64_t blocks = ((int64_t)p.max_rows * p.G + T::kRows - 1) / T::kRows;
  const int64_t most = std::max<int64_t>(1, (int64_t{1} << 22) / units);  // (a grid may have 2^32 threads)
  for (int64_t b0 = 0; b0 < blocks; b0 += most) {
    const int64_t count = std::min(most, blocks - b0);
    hipLaunchKernelGGL((paged_tile_kernel<D, QT, SIDES, Q8, WIDE>), dim3((unsigned)(units * count)), dim3(kThreads), T::kLds, stream,
                       p, (int)b0, (int)count);
  }
  return hipGetLastError();
}

template <int D, int QT, int SIDES, bool Q8>
hipError_t launch_tile(const PagedParams& p, hipStream_t stream) {
  if (1 << p.cache.page_shift >= TileTraits<D, QT, SIDES, Q8>::kStage) return launch_pages<D, QT, SIDES, Q8, true>(p, stream);
  return launch_pages<D, QT, SIDES, Q8, false>(p, stream);
}

template <int D, bool Q8>
hipError_t launch_rows(const PagedParams& p, hipStream_t stream) {
  // Two sides of 4 waves; 16 rows to a wave where those hold a request's (16 nodes of 4 heads to a key head over 32000 tokens:
  // 33.7 us, 35.9 with 32 rows), else 32 (64 nodes: 58 us, 68 with 16 rows). Heads of 192 and more, whose sums and queries would not
  // leave room for 32 rows in 256 registers (nor their stages of 64 tokens for 4 of them in LDS): 16 rows to each of 8.
  if constexpr (D > 128) return launch_tile<D, 1, 1, Q8>(p, stream);
  else if ((int64_t)p.max_rows * p.G <= 64) return launch_tile<D, 1, 2, Q8>(p, stream);
  else return launch_tile<D, 2, 2, Q8>(p, stream);
}

template <int D>
hipError_t launch_dim(const PagedParams& p, bool q8, hipStream_t stream) {
  if constexpr (D % 64 == 0) {
    if (q8) return launch_rows<D, true>(p, stream);
  }
  return launch_rows<D, false>(p, stream);
}

}  // namespace

hipError_t launch_paged_tile(const PagedParams& p, int D, bool q8, hipStream_t stream) {
  switch (D) {
    case 64: return launch_dim<64>(p, q8, stream);
    case 96: return launch_dim<96>(p, q8, stream);
    case 128: return launch_dim<128>(p, q8, stream);
    case 192: return launch_dim<192>(p, q8, stream);
    default: return launch_dim<256>(p, q8, stream);
  }
}

}  // namespace qmm4
