// Attention over pages for chunks of new tokens in bf16: tiles of 128 query rows (tokens times the query heads of a key/value head).
//
// Eight waves: four take 32 rows each over the first half of a piece's keys, four the same rows over the second half; the halves' (O, m, l) meet at
// the end.  The loop is that of the fused kernel over dense tensors (attention.hip): S^T = K.Q^T and O^T += V^T.P^T in 16 x 16 blocks of the
// bf16 MFMA, keys and values straight from memory into LDS (two K tiles and three V tiles of 64 keys per half), and the two halves one slot apart,
// so that one's products run beside the other's exponentials.  What differs:
//   - a wave fetches 16 of a block's 64 keys, which lie behind each other in a page: one page number per block and wave, out of a register that holds 64
//     blocks' numbers, a lane each; the buffer resource over them ends behind the last key that a row of the tile sees (zeros come from there);
//   - rows see keys up to their own place (and, with a window, not those too far before): blocks that some row of the wave does not see whole have their
//     scores masked;  there, where values are not all finite, the second product goes key by key, for a weight of zero would not hide them;
//   - exponentials in base 2 of s * c - m with c = scale * log2 e;
//   - work comes in pieces (attention_paged.h).
// What bounds it: the issue of MFMA and vector instructions, as there.  2048 new tokens behind 6001, 32 heads on 8 of 128 dims: 236 GFLOP in 225 to 258 us (the clock falls to 1.7 to 1.9 GHz under it),
// 0.9 to 1.05 PFLOP/s, the matrix cores busy for 48 % of the cycles: per two blocks of keys a slot of products of 1880 cycles (its 68 MFMAs take 1088) and one of exponentials of 1680, beside the other half's;
// no wave waits for memory.
// Short pieces cost more: finding the share 2.5 us, then per piece 1.5 (the tile's numbers), 2.2 (queries and pages, then keys), two slots more than blocks, and 1.3 for the meeting.  18 requests'
// single tokens and 6 chunks of 100 to 777, heads of 64 dims: 4228 blocks, 17 to a workgroup in two or three pieces, 30 us, 15 % busy; 9 requests with a window of 1024, 5 chunks, 96 dims:
// 52 us, 25 % busy.
// Tried and left: waves without a row leaving out their products (286 us for 275: the branch costs the others more); for 64 dims tiles of 64 rows, two workgroups of four waves to a compute unit
// (33.9 us where these took 31.4).
#include <algorithm>

#include "attention_paged.h"

namespace mrl {
namespace paged {
namespace {

using namespace attn;

constexpr int BKV = 64, QG = 4, BQ = 32 * QG, TH = 512;
constexpr int PRIO_A = 2, PRIO_B = 0;   // of a wave in its slot of products, of exponentials

template <int D>
struct Dims {
  static constexpr int ROW = D * 2, TILE = BKV * ROW, HALF = 5 * TILE;   // bytes of a row, of a block, of a half's tiles
  static constexpr int CHUNKS = ROW / 16, SLOTS = ROW / 32, ROWS_PER_LINE = ROW >= 256 ? 1 : 256 / ROW, ROWS_PER_LOAD = 1024 / ROW;
  static constexpr int PER_WAVE = 16 / ROWS_PER_LOAD;                    // loads of a wave's 16 keys
  static constexpr int MEET = D / 16 + 1, MERGE = 2 * QG * MEET * 1024;   // quads of a lane where the halves meet: a sixteen of rows' O, reference and denominator
  static constexpr int LDS = 2 * HALF;
  static_assert(MERGE <= LDS, "what meets at the end lies where the tiles did");
  __device__ static constexpr int k_swizzle(int row) { return (row / ROWS_PER_LINE) & (CHUNKS - 1); }
  __device__ static constexpr int v_swizzle(int row) { return (row / ROWS_PER_LINE) & (SLOTS - 1); }
};

template <int D>
__global__ __launch_bounds__(TH) void k_paged_attn(Kernargs) {
  typedef Dims<D> DD;
  constexpr int ROW = DD::ROW, TILE = DD::TILE, HALF = DD::HALF, PER_WAVE = DD::PER_WAVE;
  constexpr int NC = D / 32, NDB = D / 16, NKB = BKV / 16, NKC = BKV / 32;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qg = wave % QG, half = wave / QG;   // rows 32 qg .. of the tile; half of the keys
  const int lr = lane & 15, lgp = lane >> 4;
  uint8_t *const my_lds = lds + half * HALF;
  const uint32_t row_bytes = kernargs().p.head_dim * 2, k_slot = uint32_t(kernargs().p.key_s * 2), v_slot = uint32_t(kernargs().p.val_s * 2);

  // A load fills 1 KiB, lane l its slot l; the swizzles are applied where a lane fetches from.
  uint32_t k_src[PER_WAVE], v_src[PER_WAVE];
#pragma unroll
  for (int i = 0; i < PER_WAVE; i++) {
    const int row = i * DD::ROWS_PER_LOAD + lane / DD::CHUNKS, pc = lane % DD::CHUNKS;
    const uint32_t k_at = (pc ^ DD::k_swizzle(row)) << 4, v_at = (((pc >> 1) ^ DD::v_swizzle(row)) << 5) | ((pc & 1) << 4);
    k_src[i] = k_at < row_bytes ? row * k_slot + k_at : OUTSIDE;
    v_src[i] = v_at < row_bytes ? row * v_slot + v_at : OUTSIDE;
  }
  // Operands' addresses in a tile: of output block db and of step j these with 32 db and 64 j exclusive-ored in (rows are whole multiples of both, and tiles of 1 KiB).
  const uint32_t v_lane = (4 * lgp + (lr >> 2)) * ROW + (DD::v_swizzle(4 * lgp + (lr >> 2)) << 5) + (lr & 3) * 8;
  const uint32_t k_lane = lr * ROW + ((lgp ^ DD::k_swizzle(lr)) << 4);
  constexpr int WAIT_BUT_TWO = 0x0F70 | ((2 * PER_WAVE) & 15) | (((2 * PER_WAVE) >> 4) << 14);
  const v4i ones = {0x3f803f80, 0x3f803f80, 0x3f803f80, 0x3f803f80};
  auto mfma = [](v4i a, auto b, v4f acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), acc, 0, 0, 0);
  };

  Worker worker(kernargs());
  Piece t;
  while (worker.next(kernargs(), &t)) {
    const Kernargs &k = kernargs();
    const float c = k.c;
    const FastDiv by_group = k.by_group, by_page16 = k.by_page16;
    const uint32_t group = k.p.group, window = k.p.window;
    const float hidden = c > 0 ? -__builtin_inff() : __builtin_inff();
    const int my_blocks = int(t.b1 - t.b0), steps = (my_blocks + 1) / 2;
    const int nblocks = half ? my_blocks - steps : steps;
    const uint32_t first_block = t.begin / BKV + t.b0 + (half ? steps : 0);
    const uint8_t *const key_head = (const uint8_t *)k.p.keys + int64_t(t.head) * k.p.key_h * 2;
    const uint8_t *const val_head = (const uint8_t *)k.p.values + int64_t(t.head) * k.p.val_h * 2;
    const int64_t key_page = k.p.key_p * 2, val_page = k.p.val_p * 2;
    const int32_t *const pages = k.p.table + uint64_t(t.request) * k.p.width;
    const uint32_t page_count = k.p.pages;

    // The places of this lane's two rows (a row sees the keys up to it, below t.end and, with a window, behind it less the window; -1 where the tile
    // has no such row), and the keys that all of the wave's rows see, [all_from, all_to).
    // Q's operands go through V tiles 1 and 2 of half 1, which no fetch touches before that half's first slot of exponentials, as the lanes read them: each of the two waves that
    // have the same rows asks for a sixteen of them.
    int32_t row_at[2];
    static_assert(QG * D * 64 <= 2 * TILE, "the operands fit the two tiles");
    const uint32_t first_token = uniform(by_group.div(t.row0));
    const uint8_t *const q_first = (const uint8_t *)k.p.q + (int64_t(t.start + int32_t(first_token)) * k.p.q_t + int64_t(t.head * group) * k.p.q_h) * 2;
    const uint32_t q_lds = lds_address(lds + HALF + 3 * TILE) + qg * (2 * NC * 1024);
#pragma unroll
    for (int qb = 0; qb < 2; qb++) {
      const uint32_t i = 32 * qg + 16 * qb + lr, row = t.row0 + min(i, t.rows - 1), token = by_group.div(row), head = row - token * group;
      row_at[qb] = i < t.rows ? t.at + int32_t(token) : -1;
      if (qb == half) {
        const auto from = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(uniform(reinterpret_cast<uint64_t>(q_first))), 0, int(OUTSIDE), 0x00020000);
        const uint32_t at = ((token - first_token) * uint32_t(k.p.q_t) + head * uint32_t(k.p.q_h)) * 2;
#pragma unroll
        for (int j = 0; j < NC; j++) dma16(from, j * 64 + lgp * 16 < int(row_bytes) ? at + j * 64 + lgp * 16 : OUTSIDE, q_lds + (qb * NC + j) * 1024);
      }
    }
    const uint32_t wave_first = t.row0 + min(32u * qg, t.rows - 1), wave_last = t.row0 + min(32u * qg + 31, t.rows - 1);
    const int32_t all_to = min(t.at + int32_t(by_group.div(wave_first)) + 1, int32_t(t.end));
    const int32_t all_from = window ? int32_t(max(int64_t(t.at) + by_group.div(wave_last) - int64_t(window) + 1, int64_t(0))) : 0;
    // (that all of the tile's see)
    const int32_t tile_to = min(t.at + int32_t(first_token) + 1, int32_t(t.end));
    const int32_t tile_from = window ? int32_t(max(int64_t(t.at) + by_group.div(t.row0 + t.rows - 1) - int64_t(window) + 1, int64_t(0))) : 0;

    // Of 64 of this half's blocks, a lane each: the page of this wave's sixteen keys and the place in it, and which blocks have sixteens on no page.
    // (K runs two blocks ahead: its numbers move on before the bits of the block whose scores are masked do.)
    int32_t page_here = -1;
    uint64_t gone_here[NKB] = {}, gone_next[NKB] = {}, any_here = 0, any_next = 0;
    auto fetch_pages = [&](uint32_t kb, uint64_t *gone, uint64_t &any) {   // blocks kb .. kb + 63
      any = 0;
#pragma unroll
      for (int g = 0; g < NKB; g++) {
        const uint32_t group = (first_block + kb + lane) * 4 + g, column = by_page16.div(group);
        int32_t number = -1;
        if (int(kb) + lane < nblocks && group * 16 < t.end) {
          number = pages[column];
          if (uint32_t(number) >= page_count) number = -1;
        }
        gone[g] = __ballot(number < 0), any |= gone[g];
        if (g == qg) page_here = number;
      }
    };
    // The wave's 16 keys of a block in their page: how far behind the head's first page they begin, and the bytes from there to the end of the last one
    // that a row sees (none on no page).  Found block after block.
    struct Span {
      uint64_t keys, values;
      uint32_t key_bytes, value_bytes;
    };
    const uint32_t page_slots = k.p.page_size, place_step = uniform(BKV % page_slots);
    uint32_t place = uniform((first_block * BKV + 16 * qg) % page_slots);
    auto next_span = [&](int kb) {   // (without branches: the slot goes on beside it)
      const int32_t page = __builtin_amdgcn_readlane(page_here, kb & 63), seen = int32_t(t.end) - int32_t((first_block + kb) * BKV + 16 * qg);
      const uint32_t rows = page < 0 || kb >= nblocks ? 0 : uint32_t(min(max(seen, 0), 16));
      Span s;
      s.keys = uint64_t(uint32_t(page)) * uint32_t(key_page) + uint64_t(place * k_slot), s.key_bytes = rows ? (rows - 1) * k_slot + row_bytes : 0;
      s.values = uint64_t(uint32_t(page)) * uint32_t(val_page) + uint64_t(place * v_slot), s.value_bytes = rows ? (rows - 1) * v_slot + row_bytes : 0;
      place += place_step;
      place -= place >= page_slots ? page_slots : 0;
      return s;
    };
    auto resource = [](const uint8_t *head, uint64_t at, uint32_t bytes) {
      return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(uniform(reinterpret_cast<uint64_t>(head) + at)), 0, int(uniform(bytes)), 0x00020000);
    };
    const uint32_t k_dst0 = lds_address(my_lds) + qg * PER_WAVE * 1024, v_dst0 = k_dst0 + 2 * TILE;

    v4f o[NDB][2], den[2];
    float m_run[2] = {NO_REFERENCE, NO_REFERENCE};
#pragma unroll
    for (int qb = 0; qb < 2; qb++) {
      den[qb] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int db = 0; db < NDB; db++) o[db][qb] = v4f{0, 0, 0, 0};
    }
    // K block kb goes to K tile kb & 1, V block kb to V tile kb % 3; blocks past the half's last bring zeros to tiles that nobody reads, so that
    // every slot issues the same number of loads.  V of a block is asked for a slot after K of it, with the page that was looked up then.
    Span span = {}, span_of_v = {};   // of the block whose K is asked for last, and of the one before

    v4f s[NKB][2];
    v8bf pb[NKC][2];
    if (nblocks > 0) fetch_pages(0, gone_here, any_here);
    auto issue_k = [&](int kb) {
      span_of_v = span, span = next_span(kb);
      const auto from = resource(key_head, span.keys, span.key_bytes);
#pragma unroll
      for (int i = 0; i < PER_WAVE; i++) dma16(from, k_src[i], k_dst0 + (kb & 1) * TILE + i * 1024);
    };
    auto issue_v = [&](int kb) {   // (of the block whose K was asked for last)
      const auto from = resource(val_head, span.values, span.value_bytes);
#pragma unroll
      for (int i = 0; i < PER_WAVE; i++) dma16(from, v_src[i], v_dst0 + (kb % 3) * TILE + i * 1024);
    };
    // Before the first slot: Q and K(0), with V(0) and K(1) on their way.  Half 1 is a slot behind.
    if (nblocks > 0) {
      issue_k(0);
      issue_v(0);
      issue_k(1);
      __builtin_amdgcn_s_waitcnt(WAIT_BUT_TWO);
    } else {
      __builtin_amdgcn_s_waitcnt(0x0F70);
    }
    __syncthreads();
    v4i qf[2][NC];
#pragma unroll
    for (int qb = 0; qb < 2; qb++)
#pragma unroll
      for (int j = 0; j < NC; j++) qf[qb][j] = *(const v4i *)(lds + HALF + 3 * TILE + qg * (2 * NC * 1024) + (qb * NC + j) * 1024 + lane * 16);
    if (half) __syncthreads();
    // Where a slot's operands are: formed in the slot and not kept (the compiler would hold all of them in registers over the loop, which has none to spare).
    auto here = [&](const uint8_t *tile, uint32_t at) {
      uint32_t x = uint32_t(tile - lds) + at;
      asm volatile("" : "+v"(x));
      return x;
    };
    auto read_v = [&](uint32_t v_here, int db, int kc) {
      const uint8_t *a = lds + (v_here ^ (db << 5)) + kc * 32 * ROW;
      const v2i lo2 = read_tr16(a), hi2 = read_tr16(a + 16 * ROW);
      return v4i{lo2[0], lo2[1], hi2[0], hi2[1]};
    };
    // A slot of products: steps of two MFMAs on one operand out of LDS, which is read AHEAD steps before.
    constexpr int PV_ROWS = NDB + 1, PV_STEPS = NKC * PV_ROWS, QK_STEPS = NC * NKB, AHEAD = 2, RING = AHEAD + 1;
    v4i ring[RING];
    auto run_steps = [&](auto first_c, auto last_c, const uint8_t *lv, const uint8_t *lk) {
      constexpr int FIRST = decltype(first_c)::value, LAST = decltype(last_c)::value;
      const uint32_t v_here = here(lv, v_lane), k_here = here(lk, k_lane);
      auto fetch = [&](int x) {
        if (x < PV_STEPS) {
          if (x % PV_ROWS < NDB) ring[x % RING] = read_v(v_here, x % PV_ROWS, x / PV_ROWS);
        } else {
          ring[x % RING] = *(const v4i *)(lds + (k_here ^ ((x - PV_STEPS) / NKB << 6)) + (x - PV_STEPS) % NKB * 16 * ROW);
        }
      };
#pragma unroll
      for (int x = FIRST; x < LAST && x < FIRST + AHEAD; x++) fetch(x);
#pragma unroll
      for (int x = FIRST; x < LAST; x++) {
        if (x + AHEAD < LAST) fetch(x + AHEAD);
        const v4i a = ring[x % RING];
        if (x < PV_STEPS) {
          const int db = x % PV_ROWS, kc = x / PV_ROWS;
          if (db < NDB) {
            o[db][0] = mfma(a, pb[kc][0], o[db][0]);
            o[db][1] = mfma(a, pb[kc][1], o[db][1]);
          } else {
            den[0] = mfma(ones, pb[kc][0], den[0]);
            den[1] = mfma(ones, pb[kc][1], den[1]);
          }
        } else {
          const int kb = (x - PV_STEPS) % NKB, j = (x - PV_STEPS) / NKB;
          s[kb][0] = mfma(a, qf[0][j], s[kb][0]);
          s[kb][1] = mfma(a, qf[1][j], s[kb][1]);
        }
      }
      auto reads_group = [&](int x) {   // the builtin wants literal sizes
        if (x >= PV_STEPS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        else if (x % PV_ROWS < NDB) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      };
#pragma unroll
      for (int x = FIRST; x < LAST && x < FIRST + AHEAD; x++) reads_group(x);
#pragma unroll
      for (int x = FIRST; x < LAST; x++) {
        if (x + AHEAD < LAST) reads_group(x + AHEAD);
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      }
    };
    auto zero_s = [&]() {
#pragma unroll
      for (int kb = 0; kb < NKB; kb++) s[kb][0] = s[kb][1] = v4f{0, 0, 0, 0};
    };
    using std::integral_constant;
    // Of the block whose weights pb holds: which of its sixteens are on no page, and why some row does not see it whole: it does not see so far, or not so far back (with a window),
    // or there is a sixteen on no page; `SOME`: one of these is true for a wave of this half.
    constexpr uint32_t HIGH = 1, LOW = 2, GONE = 4, SOME = 8;
    uint32_t gone_bits = 0, masked = 0;
    // What slot B of block j wants to know is found in slot A: slot B is the longer of the two with it (2040 cycles against 1400, of 2.4 us a step; a wave issues an
    // instruction every 6 or 7 cycles there, scalar ones too).
    uint32_t masked_next = 0;
    auto prepare_pages = [&](int j) {
      if (((j + 2) & 63) == 0) fetch_pages(j + 2, gone_next, any_next);
      if ((j & 63) == 0 && j) {
        any_here = any_next;
#pragma unroll
        for (int g = 0; g < NKB; g++) gone_here[g] = gone_next[g];
      }
    };
    auto prepare = [&](int j) {
      const int32_t key0 = int32_t((first_block + j) * BKV);
      const bool gone = (any_here >> (j & 63)) & 1;
      masked_next = (key0 + BKV > all_to ? HIGH : 0) | (key0 < all_from ? LOW : 0) | (gone ? GONE : 0) | (key0 + BKV > tile_to || key0 < tile_from || gone ? SOME : 0);
      span_of_v = span, span = next_span(j + 2);
    };
    auto prepared = [&]() {   // (here, and not where it is used)
      masked_next = uniform(masked_next), span.keys = uniform(span.keys), span.key_bytes = uniform(span.key_bytes), span.values = uniform(span.values), span.value_bytes = uniform(span.value_bytes);
      asm volatile("" : "+s"(span.keys), "+s"(span.key_bytes), "+s"(masked_next), "+s"(span.values), "+s"(span.value_bytes));
    };
    // The second product of a masked block whose values are not all finite: a key at a time, its values against its weights alone, and of the product only the
    // columns (rows of queries) that see it.
    auto slow_product = [&](int kb, const uint8_t *lv) {
      const int32_t key0 = int32_t((first_block + kb) * BKV);
#pragma unroll
      for (int kc = 0; kc < NKC; kc++) {
#pragma unroll 1
        for (int x = 0; x < 32; x++) {   // key 32 kc + x: element 4 (x / 16) + x % 4 of lane group (x % 16) / 4
          const int32_t key = key0 + 32 * kc + x;
          const bool on = key < int32_t(t.end) && !((gone_bits >> (2 * kc + x / 16)) & 1);
          const bool seen0 = on && key <= row_at[0] && (!window || key > int64_t(row_at[0]) - window), seen1 = on && key <= row_at[1] && (!window || key > int64_t(row_at[1]) - window);
          const int element = 4 * (x / 16) + x % 4, bits = lgp == x % 16 / 4 ? element % 2 ? int(0xffff0000) : 0xffff : 0;
          const v4i only = {element / 2 == 0 ? bits : 0, element / 2 == 1 ? bits : 0, element / 2 == 2 ? bits : 0, element / 2 == 3 ? bits : 0};
          const uint32_t v_here = here(lv, v_lane);
          const v4i p0 = __builtin_bit_cast(v4i, pb[kc][0]) & only, p1 = __builtin_bit_cast(v4i, pb[kc][1]) & only;
#pragma unroll
          for (int db = 0; db < NDB; db++) {
            const v4i a = read_v(v_here, db, kc) & only;
            const v4f y0 = mfma(a, p0, v4f{0, 0, 0, 0}), y1 = mfma(a, p1, v4f{0, 0, 0, 0});
            o[db][0] += seen0 ? y0 : v4f{0, 0, 0, 0};
            o[db][1] += seen1 ? y1 : v4f{0, 0, 0, 0};
            asm volatile("" ::: "memory");   // (one at a time: it need not be fast, and has few registers)
          }
        }
      }
    };
    // Whether the values of a block that is masked for some wave are all finite is found in slot B, by each wave of the sixteen keys that it has fetched, and noted in the V tile that is free
    // until the next slot B: zero where they are not.
    auto note_values = [&](int vstage) {
      asm volatile("" ::: "memory");
      const uint8_t *const mine = my_lds + (2 + vstage) * TILE + qg * PER_WAVE * 1024 + lane * 16;
      uint32_t odd = 0;
#pragma unroll
      for (int i = 0; i < PER_WAVE; i++) odd |= not_finite<true>(*(const v4i *)(mine + i * 1024));
      const bool any = __any(odd != 0);
      if (lane == 0) *(int *)(my_lds + (2 + (vstage + 2) % 3) * TILE + qg * 4) = any ? 0 : 1;
    };
    // V of the block before slot j, in V tile `vstage`, for the second product.  Where the slow one has been done, zeros, in the tile with the notes (a note that another wave has
    // overwritten was one of zero, or stood beside one):
    // the fast one then adds nothing but the denominators.  (Were it left out there, its sums would be in other registers after either branch.)
    auto values_of = [&](int j, int vstage) {
      const uint8_t *const lv = my_lds + (2 + vstage) * TILE;
      if (!(masked & (HIGH | LOW | GONE))) return lv;
      uint8_t *const zeros = my_lds + (2 + (vstage + 2) % 3) * TILE;
      const v4i notes = *(const v4i *)zeros;
      if (uniform(notes[0]) && uniform(notes[1]) && uniform(notes[2]) && uniform(notes[3])) return lv;
      slow_product(j - 1, lv);
#pragma unroll 1
      for (int i = 0; i < TILE / 1024; i++) *(v4i *)(zeros + i * 1024 + lane * 16) = v4i{0, 0, 0, 0};
      return (const uint8_t *)zeros;
    };
    // Products of slot j: O += V.P of block j - 1, S = K.Q of block j; the first and the last slot have one of the two.
    auto slot_a = [&](int j, int vstage) {
      __builtin_amdgcn_s_setprio(PRIO_A);
      zero_s();
      const uint8_t *const lv = values_of(j, vstage);
      prepare_pages(j);
      prepare(j);
      run_steps(integral_constant<int, 0>{}, integral_constant<int, PV_STEPS + QK_STEPS>{}, lv, my_lds + (j & 1) * TILE);
      prepared();
    };
    auto slot_b = [&](int j, int vstage) {   // vstage: V tile of block j
      __builtin_amdgcn_s_setprio(PRIO_B);
      masked = masked_next;
      if (masked) {
        const int32_t key0 = int32_t((first_block + j) * BKV);
        if (masked & HIGH) {
#pragma unroll
          for (int qb = 0; qb < 2; qb++) {
            const int32_t last = min(row_at[qb], int32_t(t.end) - 1) - key0 - 4 * lgp;   // (of this lane's four of each sixteen)
#pragma unroll
            for (int kb = 0; kb < NKB; kb++)
#pragma unroll
              for (int r = 0; r < 4; r++) s[kb][qb][r] = kb * 16 + r > last ? hidden : s[kb][qb][r];
          }
        }
        if (masked & LOW) {
#pragma unroll
          for (int qb = 0; qb < 2; qb++) {
            const int32_t first = int32_t(max(int64_t(row_at[qb]) - window + 1, int64_t(0))) - key0 - 4 * lgp;
#pragma unroll
            for (int kb = 0; kb < NKB; kb++)
#pragma unroll
              for (int r = 0; r < 4; r++) s[kb][qb][r] = kb * 16 + r < first ? hidden : s[kb][qb][r];
          }
        }
        gone_bits = 0;
        if (masked & GONE) {
#pragma unroll
          for (int g = 0; g < NKB; g++) gone_bits |= uint32_t((gone_here[g] >> (j & 63)) & 1) << g;
#pragma unroll
          for (int kb = 0; kb < NKB; kb++)
            if ((gone_bits >> kb) & 1) s[kb][0] = s[kb][1] = v4f{hidden, hidden, hidden, hidden};
        }
      }
      auto move_reference = [&]() {
#pragma unroll
        for (int qb = 0; qb < 2; qb++) {
          float mx = s[0][qb][0] * c;
#pragma unroll
          for (int kb = 0; kb < NKB; kb++)
#pragma unroll
            for (int r = 0; r < 4; r++) mx = fmaxf(mx, s[kb][qb][r] * c);
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float m_new = fmaxf(m_run[qb], mx), alpha = __builtin_amdgcn_exp2f(m_run[qb] - m_new);
          m_run[qb] = m_new;
          den[qb] *= alpha;
#pragma unroll
          for (int db = 0; db < NDB; db++) o[db][qb] *= alpha;
        }
      };
      if (j == 0) move_reference();
      float pmax[2] = {0.0f, 0.0f};   // the block's largest exponential per row: what tells a stale reference
      // The fetches of V(j + 1) and K(j + 2) go out one at a time between the exponentials.
      const auto v_from = resource(val_head, span_of_v.values, span_of_v.value_bytes), k_from = resource(key_head, span.keys, span.key_bytes);
      const uint32_t kdst = k_dst0 + (j & 1) * TILE, vdst = v_dst0 + ((j + 1) % 3) * TILE;
#pragma unroll
      for (int kb = 0; kb < NKB; kb++)
#pragma unroll
        for (int qb = 0; qb < 2; qb++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][qb][r], c, -m_run[qb]));
            pmax[qb] = fmaxf(pmax[qb], e);
            pb[kb / 2][qb][(kb % 2) * 4 + r] = (__bf16)e;
            constexpr int EVERY = 16 / PER_WAVE;
            const int n = (kb * 2 + qb) * 4 + r;   // 0 .. 31
            if (n % EVERY == EVERY - 1) {
              const int i = n / EVERY;
              if (i < PER_WAVE) dma16(v_from, v_src[i], vdst + i * 1024);
              else dma16(k_from, k_src[i - PER_WAVE], kdst + (i - PER_WAVE) * 1024);
            }
          }
      if (j > 0 && __any(!(pmax[0] < STALE_REFERENCE) || !(pmax[1] < STALE_REFERENCE))) {
        move_reference();
#pragma unroll
        for (int qb = 0; qb < 2; qb++)
#pragma unroll
          for (int kb = 0; kb < NKB; kb++)
#pragma unroll
            for (int r = 0; r < 4; r++)
              pb[kb / 2][qb][(kb % 2) * 4 + r] = (__bf16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][qb][r], c, -m_run[qb]));
      }
      __builtin_amdgcn_s_waitcnt(WAIT_BUT_TWO);
      if (masked) note_values(vstage);
    };
    // Every wave passes steps + 1 pairs of barriers; a half with fewer blocks idles through the rest.
    if (nblocks > 0) {
      zero_s();
      prepare_pages(0);
      prepare(0);
      prepared();
      run_steps(integral_constant<int, PV_STEPS>{}, integral_constant<int, PV_STEPS + QK_STEPS>{}, my_lds, my_lds);
    }
    __syncthreads();
    if (nblocks > 0) slot_b(0, 0);
    __syncthreads();
    int vstage = 0;   // V tile of block j - 1
    for (int j = 1; j < nblocks; j++) {
      slot_a(j, vstage);
      vstage = vstage == 2 ? 0 : vstage + 1;
      __syncthreads();
      slot_b(j, vstage);
      __syncthreads();
    }
    if (nblocks > 0) run_steps(integral_constant<int, 0>{}, integral_constant<int, PV_STEPS>{}, values_of(nblocks, vstage), my_lds);
    for (int j = max(nblocks, 1); j <= steps; j++) {
      __syncthreads();
      __syncthreads();
    }
    if (!half) __syncthreads();

    // The halves meet in LDS: of the two waves that have the same rows, each puts a sixteen of them together.  The fetches past the last block must not land there.
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    v4f *const given = (v4f *)lds + wave * (DD::MEET * 64) + lane;
    const v4f *const taken = (const v4f *)lds + (wave ^ QG) * (DD::MEET * 64) + lane;
#pragma unroll
    for (int db = 0; db < NDB; db++) given[db * 64] = half ? o[db][0] : o[db][1];
    given[NDB * 64] = half ? v4f{m_run[0], den[0][0], 0, 0} : v4f{m_run[1], den[1][0], 0, 0};
    __syncthreads();
    const Kernargs &e = kernargs();
    const bool whole = t.whole();
    if (!whole && t.b0 == 0) {
      worker.described = true;
      if (tid == 0) worker.describe(e.w, t);
    }
    const uint32_t i = 32 * qg + 16 * half + lr;
    if (i < t.rows) {
      const v4f ml = taken[NDB * 64];
      const float m_own = half ? m_run[1] : m_run[0], mm = fmaxf(m_own, ml[0]);
      float own = __builtin_amdgcn_exp2f(m_own - mm), other = __builtin_amdgcn_exp2f(ml[0] - mm);
      const float l = (half ? den[1][0] : den[0][0]) * own + ml[1] * other;
      if (!whole) {
        float *const to = worker.place(e.w, t, BQ * (D + 4)) + i * (D + 4);
#pragma unroll
        for (int db = 0; db < NDB; db++) *(v4f *)(to + db * 16 + 4 * lgp) = (half ? o[db][1] : o[db][0]) * own + taken[db * 64] * other;
        if (lgp == 0) to[D] = mm, to[D + 1] = l;
      } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        own *= inv, other *= inv;
        const uint32_t row = t.row0 + i, token = e.by_group.div(row), head = t.head * e.p.group + (row - token * e.p.group);
        __bf16 *out = (__bf16 *)e.p.out + int64_t(t.start + int32_t(token)) * e.p.o_t + int64_t(head) * e.p.o_h;
        typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int db = 0; db < NDB; db++) {
          const v4f v = (half ? o[db][1] : o[db][0]) * own + taken[db * 64] * other;
          const uint32_t dim = db * 16 + 4 * lgp;
          if (dim < e.p.head_dim) *(v4bf *)(out + dim) = v4bf{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        }
      }
    }
    __syncthreads();   // (the next piece's tiles come where the halves met)
  }
  if (tid == 0 && !worker.described) kernargs().w.merges[worker.number * 8] = 0;
}

template <int D>
hipError_t launch_one(const PagedAttnArgs &a, Work work, hipStream_t stream) {
  constexpr int LDS = Dims<D>::LDS;
  static std::atomic<uint64_t> lds_limit_set{0};
  if (!plan::recording()) {
    const hipError_t e = raise_lds_limit(lds_limit_set, (const void *)k_paged_attn<D>, LDS);
    if (e != hipSuccess) return e;
  }
  plan::work(plan::UNIT_MFMA_BF16, 4.0 * a.tokens * a.q_heads * D * double(a.width) * a.page_size,
             4.0 * a.kv_heads * a.head_dim * double(a.width) * a.page_size * a.requests + 4.0 * a.tokens * double(a.q_heads) * a.head_dim);
  MRL_LAUNCH(k_paged_attn<D>, dim3(work.workers), dim3(TH), LDS, stream, Kernargs{a, work, FastDiv(a.group), FastDiv(a.page_size / 16), a.scale * LOG2E});
  return plan::last_error();
}

}  // namespace

void chunk_work(const PagedAttnArgs &a, Work *w) {
  w->workers = g_compute_units;   // (one of D = 128 to a compute unit's LDS)
  // us, recorded into a graph; cases that are not named are within 1 %.
  //   least 4, 8, 16: 5 requests, 2 chunks to 300, 64 dims 18.8, 19.7, 17.7; 200 new tokens behind 3000, 128 dims 46.5, 46.4, 45.5
  //   overhead 4, 7, 11 of 64 dims: the mixed batch 36.9, 34.0, 34.6; 2, 4, 8 of 128: the window's 57.0, 54.9, 57.0, 2048 tokens behind 6001 248, 244, 244
  //   second 0, 7, 16: the first two 17.7, 19.7, 19.9 and 45.5, 46.4, 46.5
  w->bq_log2 = 7, w->block_log2 = 6, w->least = 8, w->overhead = a.head_dim <= 64 ? 7 : 4, w->second = 7;
}

hipError_t launch_chunk(const PagedAttnArgs &a, const Work &work, hipStream_t stream) {
  return a.head_dim <= 64 ? launch_one<64>(a, work, stream) : launch_one<128>(a, work, stream);
}

}  // namespace paged
}  // namespace mrl
