// Attention over pages with the KEYS dealt to the waves of a workgroup: for few query rows per request (a decoding step, some tokens at once)
// and for f32.
//
// A workgroup owns a piece of a tile (attention_paged.h) of 16 * QB rows; each of its W waves takes every W-th block of 32 keys, and the waves'
// (O, m, l) meet at the end in LDS.  Both products are formed transposed, in blocks of 16 x 16: S^T = K.Q^T, O^T += V^T.P^T, so that
// a lane owns a query row (l % 16 of the block's columns): running reference, denominator and rescaling are its scalars.  The index that
// a product sums over may be dealt to lanes in any order that both operands share: lane group g = l / 16 holds keys 4 g .. 4 g + 3 of each 16
// in its accumulators of the first product, and these are the operand of the second as they stand.
//   bf16: v_mfma 16x16x32; V's operand through the transposing read; P rounded to bf16 (2^-8), the denominators from a row of ones, so that
//         they are the sums of the very numbers that weigh the values.  (The second product in f32 would take 16 times the matrix cores' time.  Error against 64 bits, root mean
//         square over root mean square: 0.0017 of the result's own rounding alone, 0.0017 to 0.0022 with this one, most over 130001 keys.)
//   f32:  v_mfma 16x16x4; a 16-byte read of a K row is four steps of dims, a V row is read in words.  The matrix cores bound it (1/16 of bf16's rate), so
//         there are forms for 80 and 96 dims, too, and a tile of up to 16 rows does half of a form of 32.
// Keys and values go from their pages straight into LDS, 16 bytes a lane, through a buffer resource per 16 keys: a page's numbers are whole sixteens of
// slots, so 16 keys lie behind each other.  The resource ends behind the last key that a row of the tile sees: what lies behind (or on no
// page at all) arrives as zeros, whatever the slots hold.  The pages' numbers are fetched 32 blocks at a time, a lane each, and read from
// the lanes.
//
// Exponentials are taken in base 2 of s * c - m, c = scale * log2 e; the reference m is the row's largest score so far in the first
// blocks, and moves later only when a score has outgrown it by 2^40.
//
// What bounds it, in bf16: memory.  48 requests of 300 to 16384 keys, 8 heads of 128 dims, one new token each: 810 MB in 136 us, 5.9 TB/s (all that memory delivers is those bytes: FETCH_SIZE counts
// 809.7 MB); one of 130001 keys 532 MB in 87 us, 6.1 TB/s.  Without `nt` on the loads of what is read once the first takes 157 us.  Two or four workgroups of four waves to a compute
// unit, each wave with a block of K and one of V in flight, keep 128 KB of a compute unit's LDS filling.  4 requests up to 564 keys, 16 heads, a workgroup each: 10 us, eight rounds of a trip
// to memory (four waves instead of eight: 11.8).  f32, 5 requests, 12 heads of 80 dims, 3 chunks of 33 to 260 tokens up to 1501 keys: 24.5 us, of which the matrix cores are busy for 4
// and what a share costs before its first product (4 us), its first fetch and the meeting take most; with products over 128 dims and 32 rows always it took 35.
#include <algorithm>

#include "attention_paged.h"

namespace mrl {
namespace paged {
namespace {

using namespace attn;

constexpr int KEYS = 32;      // keys per block
constexpr int WAVES = 4;      // of a workgroup; where it has a head of a request to itself and LDS allows, twice as many
constexpr int FOLLOWED = 4;   // blocks of a wave whose maxima the reference follows

template <class T, int D, int QB, int W>
struct Form {
  static constexpr bool BF16 = sizeof(T) == 2;
  static constexpr int TH = 64 * W, BQ = 16 * QB;
  static constexpr int ROW = D * int(sizeof(T)), CHUNKS = ROW / 16, SLOTS = ROW / 32;
  static constexpr int TILE = KEYS * ROW, LOADS = TILE / 1024, HALF = LOADS / 2;
  static constexpr int ROWS_PER_LINE = ROW >= 256 ? 1 : 256 / ROW;   // rows per 256-byte line of banks
  static constexpr int NDB = D / 16;                                  // 16-row blocks of O^T
  static constexpr int ROW_FLOATS = D + 4;                            // of a partial result: O, reference, denominator
  static_assert(16 * ROW % 1024 == 0 && LOADS < 64, "16 keys are whole loads");
  // K rows of 2^n bytes are XOR-swizzled by 16-byte chunk, bf16's V rows by 32-byte slot (attention_keys.hip); the others lie as they are: 16 lanes read 16 words of
  // an f32 row of V, and what meets in the banks by that is read while the products are busy.
  __device__ static constexpr int k_swizzle(int row) { return CHUNKS & (CHUNKS - 1) ? 0 : (row / ROWS_PER_LINE) & (CHUNKS - 1) & 15; }
  __device__ static constexpr int v_swizzle(int row) { return BF16 ? (row / ROWS_PER_LINE) & (SLOTS - 1) & 15 : 0; }
  // The waves' tiles, or after the loop their O, references and denominators.
  static constexpr int TILES = W * 2 * TILE, TRIPLES = W * (QB * D * 64 + QB * 128);
  static constexpr int LDS = TILES > TRIPLES ? TILES : TRIPLES;
  // Waves of a SIMD, and workgroups of a compute unit, by LDS and by registers.
  static constexpr int BY_LDS = 160 * 1024 / LDS * W / 4, ON_SIMD = BY_LDS >= 4 && QB == 1 ? 4 : BY_LDS >= 2 ? 2 : 1, RESIDENT = ON_SIMD * 4 / W;
};

__device__ inline float over_lane_groups(float x) {   // the largest over the four lane groups, in all of them
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}

// The head dim may be below D, in whole 16-byte chunks: zeros behind it.
template <class T, int D, int QB, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(Form<T, D, QB, W>::ON_SIMD))) void k_paged_attn(Kernargs) {
  using F = Form<T, D, QB, W>;
  constexpr bool BF16 = F::BF16;
  constexpr int ROW = F::ROW, TILE = F::TILE, LOADS = F::LOADS, HALF = F::HALF, NDB = F::NDB;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lgp = lane >> 4;
  uint8_t *const k_tile = lds + wave * 2 * TILE, *const v_tile = k_tile + TILE;
  const uint32_t row_bytes = kernargs().p.head_dim * uint32_t(sizeof(T)), k_slot = uint32_t(kernargs().p.key_s * sizeof(T)), v_slot = uint32_t(kernargs().p.val_s * sizeof(T));

  // One instruction fills 1 KiB of a tile, lane l its slot l: row and chunk that belong there.  The second 16 keys are as the first, from their
  // own base.
  uint32_t k_src[HALF], v_src[HALF];
  {
#pragma unroll
    for (int i = 0; i < HALF; i++) {
      const int row = (i * 64 + lane) / F::CHUNKS, ld_pc = (i * 64 + lane) % F::CHUNKS;
      const uint32_t k_at = (ld_pc ^ F::k_swizzle(row)) << 4;
      const uint32_t v_at = BF16 ? (((ld_pc >> 1) ^ F::v_swizzle(row)) << 5) | ((ld_pc & 1) << 4) : ld_pc << 4;
      k_src[i] = k_at < row_bytes ? row * k_slot + k_at : OUTSIDE;
      v_src[i] = v_at < row_bytes ? row * v_slot + v_at : OUTSIDE;
    }
  }
  const uint32_t k_dst = lds_address(k_tile), v_dst = lds_address(v_tile);
  // Lane-dependent parts of the operands' addresses.
  constexpr int NC = D * int(sizeof(T)) / 64;   // 64-byte pieces of a K row: bf16 a step of 32 dims, f32 four steps of 4
  uint32_t k_lane[NC], v_lane[NDB];
#pragma unroll
  for (int i = 0; i < NC; i++) k_lane[i] = lr * ROW + (((4 * i + lgp) ^ F::k_swizzle(lr)) << 4);
#pragma unroll
  for (int i = 0; i < NDB; i++) {
    const int vrow = 4 * lgp + (lr >> 2);
    v_lane[i] = BF16 ? vrow * ROW + ((i ^ F::v_swizzle(vrow)) << 5) + (lr & 3) * 8 : 4 * lgp * ROW + i * 64 + lr * 4;
  }
  constexpr int ALL_BUT_ONE_TILE = 0x0F70 | (LOADS & 15) | ((LOADS >> 4) << 14), ALL = 0x0F70, READS_DONE = 0xC07F;

  const bool direct = kernargs().w.direct;
  // NQ: of the QB columns of 16 rows, those that the tile has rows in.
  auto run = [&](auto columns, const Kernargs &k, const Piece &t, Worker *worker) {
    constexpr int NQ = decltype(columns)::value;
    const float c = k.c;
    const FastDiv by_group = k.by_group, by_page16 = k.by_page16;
    const uint32_t group = k.p.group, window = k.p.window, first_block = t.begin / KEYS + t.b0 + wave;
    const bool once = k.w.once;
    const float hidden = c > 0 ? -__builtin_inff() : __builtin_inff();   // a score that weighs nothing

    // This lane's rows: queries, and the keys they see, [lo, hi].
    v4i qf[NQ][NC];
    int32_t lo[NQ], hi[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; qb++) {
      const uint32_t i = 16 * qb + lr, row = t.row0 + min(i, t.rows - 1), token = by_group.div(row), head = t.head * group + (row - token * group);
      const int32_t at = t.at + int32_t(token);
      hi[qb] = i < t.rows ? min(at, int32_t(t.end) - 1) : -1;
      lo[qb] = window ? int32_t(max(int64_t(at) - int64_t(window) + 1, int64_t(0))) : 0;
      const uint8_t *q = (const uint8_t *)k.p.q + (int64_t(t.start + int32_t(token)) * k.p.q_t + int64_t(head) * k.p.q_h) * int64_t(sizeof(T));
#pragma unroll
      for (int j = 0; j < NC; j++) {
        const uint32_t from = j * 64 + lgp * 16;
        qf[qb][j] = from < row_bytes ? *(const v4i *)(q + from) : v4i{0, 0, 0, 0};
      }
    }
    // Blocks that every row sees whole lie in [all_from, all_to).
    const int32_t first_at = t.at + int32_t(by_group.div(t.row0)), last_at = t.at + int32_t(by_group.div(t.row0 + t.rows - 1));
    const int32_t all_to = min(first_at + 1, int32_t(t.end));
    const int32_t all_from = window ? int32_t(max(int64_t(last_at) - int64_t(window) + 1, int64_t(0))) : 0;

    // The pages' numbers of 32 of this wave's blocks, both sixteens of each, one a lane, and the places in the page.
    int32_t page_here = -1;
    uint32_t place_here = 0;
    const int32_t *const pages = k.p.table + uint64_t(t.request) * k.p.width;
    const uint32_t page_count = k.p.pages, groups_per_page = k.p.page_size / 16;
    auto fetch_pages = [&](uint32_t n) {   // of the wave's blocks n .. n + 31
      const uint32_t mine = n + (lane >> 1), group16 = (first_block + mine * W) * 2 + (lane & 1), column = by_page16.div(group16);
      page_here = -1, place_here = (group16 - column * groups_per_page) * 16;
      if (t.b0 + wave + mine * W < t.b1 && group16 * 16 < t.end) {
        const int32_t number = pages[column];
        if (uint32_t(number) < page_count) page_here = number;
      }
    };
    // Of the wave's n-th block, 16 keys each: through a resource that ends behind the last one that a row sees.
    auto page_of = [&](uint32_t n, int half) { return __builtin_amdgcn_readlane(page_here, (n & 31) * 2 + half); };
    auto issue = [&](uint32_t n, const uint8_t *head, int64_t page_bytes, uint32_t slot_bytes, const uint32_t *src, uint32_t dst) {
      const uint32_t key0 = (first_block + n * W) * KEYS;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int32_t page = page_of(n, half);
        const uint32_t place = __builtin_amdgcn_readlane(place_here, (n & 31) * 2 + half), from = key0 + 16 * half;
        const uint32_t rows = page < 0 || from >= t.end ? 0 : min(t.end - from, 16u);
        const uint64_t base = reinterpret_cast<uint64_t>(head) + uint64_t(max(page, 0)) * page_bytes + uint64_t(place) * slot_bytes;
        const auto from_buf = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(uniform(base)), 0, uniform(int(rows ? (rows - 1) * slot_bytes + row_bytes : 0)), 0x00020000);
        if (once) {
#pragma unroll
          for (int i = 0; i < HALF; i++) dma16_once(from_buf, src[i], dst + (half * HALF + i) * 1024);
        } else {
#pragma unroll
          for (int i = 0; i < HALF; i++) dma16_ordered(from_buf, src[i], dst + (half * HALF + i) * 1024);
        }
      }
    };
    const uint8_t *const key_head = (const uint8_t *)k.p.keys + int64_t(t.head) * k.p.key_h * int64_t(sizeof(T));
    const uint8_t *const val_head = (const uint8_t *)k.p.values + int64_t(t.head) * k.p.val_h * int64_t(sizeof(T));
    const int64_t key_page = k.p.key_p * int64_t(sizeof(T)), val_page = k.p.val_p * int64_t(sizeof(T));
    auto issue_k = [&](uint32_t n) { issue(n, key_head, key_page, k_slot, k_src, k_dst); };
    auto issue_v = [&](uint32_t n) { issue(n, val_head, val_page, v_slot, v_src, v_dst); };

    v4f o[NDB][NQ], den[NQ];
    float m_run[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; qb++) {
      m_run[qb] = NO_REFERENCE;
      den[qb] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int db = 0; db < NDB; db++) o[db][qb] = v4f{0, 0, 0, 0};
    }
    auto mfma16 = [](v4i a, auto b, v4f acc) {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), acc, 0, 0, 0);
    };
    auto mfma4 = [](float a, float b, v4f acc) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, acc, 0, 0, 0); };

    // This wave's blocks: t.b0 + wave, + W, ..
    const uint32_t mine = t.b1 - t.b0 > uint32_t(wave) ? (t.b1 - t.b0 - wave + W - 1) / W : 0;
    if (mine) {
      fetch_pages(0);
      issue_k(0);
      issue_v(0);
      bool start = true;
      __builtin_amdgcn_s_waitcnt(ALL);
      for (uint32_t n = 0; n < mine; n++) {
        const bool more = n + 1 < mine;
        // In flight at this point, oldest first: K of this block, V of this block.
        if (!start) __builtin_amdgcn_s_waitcnt(ALL_BUT_ONE_TILE);
        asm volatile("" ::: "memory");
        v4f s[2][NQ];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
#pragma unroll
          for (int qb = 0; qb < NQ; qb++) s[kb][qb] = v4f{0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < NC; j++) {
            const v4i a = *(const v4i *)(k_tile + k_lane[j] + kb * 16 * ROW);
#pragma unroll
            for (int qb = 0; qb < NQ; qb++) {
              if constexpr (BF16) {
                s[kb][qb] = mfma16(a, qf[qb][j], s[kb][qb]);
              } else {
#pragma unroll
                for (int r = 0; r < 4; r++) s[kb][qb] = mfma4(__int_as_float(a[r]), __int_as_float(qf[qb][j][r]), s[kb][qb]);
              }
            }
          }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(READS_DONE);   // K's operands are in registers: its tile may be filled again
        const bool gone0 = page_of(n, 0) < 0, gone1 = page_of(n, 1) < 0;
        if (more) {
          if (((n + 1) & 31) == 0) fetch_pages(n + 1);
          issue_k(n + 1);
        }
        const int32_t key0 = int32_t((first_block + n * W) * KEYS);
        const bool masked = key0 < all_from || key0 + KEYS > all_to || gone0 || gone1;
        if (masked) {
#pragma unroll
          for (int qb = 0; qb < NQ; qb++) {
            const int32_t last = hi[qb] - key0 - 4 * lgp, first = lo[qb] - key0 - 4 * lgp;   // (of this lane's four of each sixteen)
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
              for (int r = 0; r < 4; r++) s[kb][qb][r] = kb * 16 + r > last || kb * 16 + r < first || (kb ? gone1 : gone0) ? hidden : s[kb][qb][r];
          }
        }
        auto move_reference = [&]() {
#pragma unroll
          for (int qb = 0; qb < NQ; qb++) {
            float mx = s[0][qb][0] * c;
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
              for (int r = 0; r < 4; r++) mx = fmaxf(mx, s[kb][qb][r] * c);
            mx = over_lane_groups(mx);
            const float m_new = fmaxf(m_run[qb], mx);
            const float alpha = __builtin_amdgcn_exp2f(m_run[qb] - m_new);
            m_run[qb] = m_new;
            den[qb] *= alpha;
#pragma unroll
            for (int db = 0; db < NDB; db++) o[db][qb] *= alpha;
          }
        };
        const bool fresh = n < FOLLOWED;
        float e[2][NQ][4];
        float pmax = 0.0f;
        auto exponentials = [&]() {
#pragma unroll
          for (int qb = 0; qb < NQ; qb++)
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
              for (int r = 0; r < 4; r++) {
                e[kb][qb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][qb][r], c, -m_run[qb]));
                pmax = fmaxf(pmax, e[kb][qb][r]);
              }
        };
        if (fresh) move_reference();
        exponentials();
        if (!fresh && __any(!(pmax < STALE_REFERENCE))) {
          move_reference();
          exponentials();
        }
        start = false;
        v8bf pb[NQ];
        if constexpr (BF16) {
#pragma unroll
          for (int qb = 0; qb < NQ; qb++)
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
              for (int r = 0; r < 4; r++) pb[qb][kb * 4 + r] = (__bf16)e[kb][qb][r];
        }
        if (more) __builtin_amdgcn_s_waitcnt(ALL_BUT_ONE_TILE);   // V of this block is in; K of the next may still be under way
        else __builtin_amdgcn_s_waitcnt(ALL);
        asm volatile("" ::: "memory");
        uint32_t odd = 0;   // a value that is not finite, in a block that not every row sees whole: a weight of zero would not hide it
        if (masked) {
#pragma unroll
          for (int i = 0; i < TILE / 1024; i++) odd |= not_finite<BF16>(*(const v4i *)(v_tile + i * 1024 + lane * 16));
        }
        if (__any(odd != 0)) {
          // A key at a time, its values against its weights alone, and of the product only the columns (query rows) that see it.
          if constexpr (BF16) {
#pragma unroll 1
            for (int x = 0; x < KEYS; x++) {   // element 4 (x / 16) + x % 4 of lane group (x % 16) / 4
              const int element = 4 * (x / 16) + x % 4, bits = lgp == x % 16 / 4 ? element % 2 ? int(0xffff0000) : 0xffff : 0;
              const v4i only = {element / 2 == 0 ? bits : 0, element / 2 == 1 ? bits : 0, element / 2 == 2 ? bits : 0, element / 2 == 3 ? bits : 0};
#pragma unroll
              for (int db = 0; db < NDB; db++) {
                const v2i lo2 = read_tr16(v_tile + v_lane[db]), hi2 = read_tr16(v_tile + v_lane[db] + 16 * ROW);
                const v4i a = v4i{lo2[0], lo2[1], hi2[0], hi2[1]} & only;
#pragma unroll
                for (int qb = 0; qb < NQ; qb++) {
                  const v4f y = mfma16(a, __builtin_bit_cast(v4i, pb[qb]) & only, v4f{0, 0, 0, 0});
                  o[db][qb] += key0 + x >= lo[qb] && key0 + x <= hi[qb] && !(x < 16 ? gone0 : gone1) ? y : v4f{0, 0, 0, 0};
                }
                asm volatile("" ::: "memory");   // (one at a time: it need not be fast, and has few registers)
              }
            }
          } else {
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
              for (int r = 0; r < 4; r++)
#pragma unroll 1
                for (int g = 0; g < 4; g++) {
                  const int32_t key = key0 + kb * 16 + 4 * g + r;
#pragma unroll
                  for (int db = 0; db < NDB; db++) {
                    const float a = *(const float *)(v_tile + v_lane[db] + (kb * 16 + r) * ROW);
#pragma unroll
                    for (int qb = 0; qb < NQ; qb++) {
                      const v4f y = mfma4(lgp == g ? a : 0.0f, lgp == g ? e[kb][qb][r] : 0.0f, v4f{0, 0, 0, 0});
                      o[db][qb] += key >= lo[qb] && key <= hi[qb] && !(kb ? gone1 : gone0) ? y : v4f{0, 0, 0, 0};
                    }
                    asm volatile("" ::: "memory");
                  }
                }
          }
          // What is left of the block are its denominators: the product below adds zeros.
#pragma unroll 1
          for (int i = 0; i < TILE / 1024; i++) *(v4i *)(v_tile + i * 1024 + lane * 16) = v4i{0, 0, 0, 0};
        }
        if constexpr (BF16) {
#pragma unroll
          for (int db = 0; db < NDB; db++) {
            const v2i lo2 = read_tr16(v_tile + v_lane[db]), hi2 = read_tr16(v_tile + v_lane[db] + 16 * ROW);
            const v4i a = {lo2[0], lo2[1], hi2[0], hi2[1]};
#pragma unroll
            for (int qb = 0; qb < NQ; qb++) o[db][qb] = mfma16(a, pb[qb], o[db][qb]);
          }
        } else {
#pragma unroll
          for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
              for (int db = 0; db < NDB; db++) {
                const float a = *(const float *)(v_tile + v_lane[db] + (kb * 16 + r) * ROW);
#pragma unroll
                for (int qb = 0; qb < NQ; qb++) o[db][qb] = mfma4(a, e[kb][qb][r], o[db][qb]);
              }
        }
        if constexpr (BF16) {
          const v4i ones = {0x3f803f80, 0x3f803f80, 0x3f803f80, 0x3f803f80};
#pragma unroll
          for (int qb = 0; qb < NQ; qb++) den[qb] = mfma16(ones, pb[qb], den[qb]);
        } else {
#pragma unroll
          for (int qb = 0; qb < NQ; qb++)
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
              for (int r = 0; r < 4; r++) den[qb][r] += e[kb][qb][r];
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(READS_DONE);
        if (more) issue_v(n + 1);
      }
    }

    // The waves' triples meet: quads of O in LDS as [wave][block column][quad][lane], then [wave][block column][reference, denominator][row].
    // Quad x of a lane holds dims 16 x + 4 lgp .. + 3.
    __syncthreads();   // all tiles have been read
    v4f *const quads = (v4f *)lds;
    float *const stats = (float *)(lds + W * NQ * D * 64);
#pragma unroll
    for (int qb = 0; qb < NQ; qb++) {
#pragma unroll
      for (int x = 0; x < NDB; x++) quads[((wave * NQ + qb) * NDB + x) * 64 + lane] = o[x][qb];
      float l = den[qb][0];
      if constexpr (!BF16) {
        l = (den[qb][0] + den[qb][1]) + (den[qb][2] + den[qb][3]);
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
      }
      if (lgp == 0) stats[(wave * NQ + qb) * 32 + lr] = m_run[qb], stats[(wave * NQ + qb) * 32 + 16 + lr] = l;
    }
    __syncthreads();
    const Kernargs &e = kernargs();
    const bool whole = t.whole();
    float *const part = whole ? nullptr : worker->place(e.w, t, F::BQ * F::ROW_FLOATS);
    if (!whole && t.b0 == 0) {
      worker->described = true;
      if (tid == 0) worker->describe(e.w, t);
    }
#pragma unroll
    for (int x0 = 0; x0 < NQ * NDB; x0 += W) {
      const int x = x0 + wave, qb = x / NDB;
      if (NQ * NDB % W && x >= NQ * NDB) break;
      const uint32_t i = 16 * qb + lr;
      if (i >= t.rows) continue;
      float mm = -3.0e38f, l = 0.0f;
      float f[W];
#pragma unroll
      for (int j = 0; j < W; j++) f[j] = stats[(j * NQ + qb) * 32 + lr], mm = fmaxf(mm, f[j]);
      v4f sum = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < W; j++) {
        f[j] = __builtin_amdgcn_exp2f(f[j] - mm);
        l += stats[(j * NQ + qb) * 32 + 16 + lr] * f[j];
        sum += quads[((j * NQ + qb) * NDB + x % NDB) * 64 + lane] * f[j];
      }
      const uint32_t dim = x % NDB * 16 + 4 * lgp;
      if (!whole) {
        float *to = part + i * F::ROW_FLOATS;
        *(v4f *)(to + dim) = sum;
        if (dim == 0) to[D] = mm, to[D + 1] = l;
        continue;
      }
      if (dim >= e.p.head_dim) continue;
      sum *= l == 0.0f ? 0.0f : 1.0f / l;
      const uint32_t row = t.row0 + i, token = e.by_group.div(row), head = t.head * e.p.group + (row - token * e.p.group);
      T *out = (T *)e.p.out + int64_t(t.start + int32_t(token)) * e.p.o_t + int64_t(head) * e.p.o_h + dim;
      if constexpr (BF16) {
        typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
        *(v4bf *)out = v4bf{(__bf16)sum[0], (__bf16)sum[1], (__bf16)sum[2], (__bf16)sum[3]};
      } else {
        *(v4f *)out = sum;
      }
    }
  };
  auto run_piece = [&](const Kernargs &k, const Piece &t, Worker *worker) {
    if constexpr (!BF16 && QB > 1) {
      if (t.rows <= 16) return run(std::integral_constant<int, 1>{}, k, t, worker);
    }
    run(std::integral_constant<int, QB>{}, k, t, worker);
  };
  Piece t;
  if (direct) {
    DirectWorker worker(kernargs());
    while (worker.next(kernargs(), &t)) {
      run_piece(kernargs(), t, nullptr);
      __syncthreads();   // (the triples have been read)
    }
    return;
  }
  Worker worker(kernargs());
  while (worker.next(kernargs(), &t)) {
    run_piece(kernargs(), t, &worker);
    __syncthreads();   // (the triples have been read)
  }
  if (tid == 0 && !worker.described) kernargs().w.merges[worker.number * 8] = 0;
}

template <class T, int D, int QB, int W>
hipError_t launch_one(const PagedAttnArgs &a, Work work, hipStream_t stream) {
  using F = Form<T, D, QB, W>;
  static std::atomic<uint64_t> lds_limit_set{0};
  if (!plan::recording()) {
    const hipError_t e = raise_lds_limit(lds_limit_set, (const void *)k_paged_attn<T, D, QB, W>, F::LDS);
    if (e != hipSuccess) return e;
  }
  const uint32_t grid = work.direct ? a.requests * a.kv_heads : work.workers;
  const double keys = double(a.width) * a.page_size * a.requests;   // (all that the table holds: the lengths are on the device)
  plan::work(F::BF16 ? plan::UNIT_MFMA_BF16 : plan::UNIT_MFMA_F32, 4.0 * a.tokens * a.q_heads * D * double(a.width) * a.page_size,
             2.0 * sizeof(T) * a.kv_heads * a.head_dim * keys + 2.0 * sizeof(T) * a.tokens * double(a.q_heads) * a.head_dim);
  MRL_LAUNCH((k_paged_attn<T, D, QB, W>), dim3(grid), dim3(F::TH), F::LDS, stream, Kernargs{a, work, FastDiv(a.group), FastDiv(a.page_size / 16), a.scale * LOG2E});
  return plan::last_error();
}

// Calls f with the form's types and sizes.
template <class T, int D, class F>
auto with_rows(int qb, bool direct, F f) {
  constexpr int MORE = Form<T, D, 1, 2 * WAVES>::LDS <= 160 * 1024 ? 2 * WAVES : WAVES;
  if (direct) return qb == 1 ? f(Form<T, D, 1, MORE>()) : f(Form<T, D, 2, MORE>());
  return qb == 1 ? f(Form<T, D, 1, WAVES>()) : f(Form<T, D, 2, WAVES>());
}
template <class F>
auto with_form(const PagedAttnArgs &a, int qb, bool direct, F f) {
  if (a.dtype == MRL_BF16) return a.head_dim <= 64 ? with_rows<__bf16, 64>(qb, direct, f) : with_rows<__bf16, 128>(qb, direct, f);
  if (a.head_dim <= 64) return with_rows<float, 64>(qb, direct, f);
  if (a.head_dim <= 80) return with_rows<float, 80>(qb, direct, f);
  return a.head_dim <= 96 ? with_rows<float, 96>(qb, direct, f) : with_rows<float, 128>(qb, direct, f);
}
template <class T, int D, int QB, int W>
hipError_t launch_form(Form<T, D, QB, W>, const PagedAttnArgs &a, const Work &work, hipStream_t stream) {
  return launch_one<T, D, QB, W>(a, work, stream);
}
}  // namespace

void keys_work(const PagedAttnArgs &a, int qb, Work *w) {
  // us, recorded into a graph; cases that are not named are within 1 %.
  //   least 2, 4, 8: 4 requests to 564 keys, 16 heads, in wide tables 13.9, 14.4, 16.3; one of 8000 keys, 2 heads 18.3, 17.2, 17.3; 4 requests of 6 new tokens to 2000 keys 32.2, 29.5, 31.8
  //   overhead 1, 3, 8: 16 requests of 3 new tokens to 16384 keys, 8 heads 76.2, 79.1, 79.2; 48 single tokens' 146.1, 146.6, 147.9
  //   second 4, 12, 24: the first of these 75.7, 79.1, 79.0
  w->workers = g_compute_units * with_form(a, qb, false, [](auto f) { return uint32_t(decltype(f)::RESIDENT); });
  w->bq_log2 = qb == 1 ? 4 : 5, w->block_log2 = 5, w->least = WAVES, w->overhead = 3, w->second = 3 * WAVES;
}

hipError_t launch_keys(const PagedAttnArgs &a, const Work &work, int qb, hipStream_t stream) {
  return with_form(a, qb, work.direct, [&](auto f) { return launch_form(f, a, work, stream); });
}

}  // namespace paged
}  // namespace mrl
