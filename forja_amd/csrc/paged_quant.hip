// The paged key/value cache held in 8 bits: storing rows, reading them back, and ragged attention over it.
//
// A row (one token, one kv head) is held as e4m3 codes c_i and one power of two 2^e:
//   e   = the smallest whole number with max |x_i| <= 448 * 2^e over the row's finite x_i, at least -126
//   c_i = x_i / 2^e rounded to e4m3, ties to even (x_i that is not finite: the code of no number)
// and stands for c_i * 2^e.  Codes are [pages, page_tokens, heads, width] bytes, scales the byte e + 127 in
// [pages, 2 (keys, values), heads, page_tokens rounded up to 4]; a zero byte stands for a row of zeros, as
// fresh storage reads.  Why a power of two: a floating code's relative step is the same over its whole range, so
// another factor gains nothing, x_i / 2^e is exact (a code is rounded once), and the byte is what the matrix
// cores' scaled products take.  Why a scale for every token: storing a row never changes what is stored already,
// so a cache does not depend on how its sequence was cut into chunks, and shared pages stay what they are.
#include <algorithm>
#include <atomic>

#include "fast_kernels.hpp"
#include "paged_common.hpp"

namespace fh {

namespace {

typedef __attribute__((ext_vector_type(2))) float f32x2;

constexpr uint32_t kWordsHeld = 2;   // code words of a row that a lane holds: rows of up to 512 values

// Scale byte of a row whose largest finite magnitude is `most`.
__device__ inline uint32_t scale_byte(float most) {
  const uint32_t exponent = (__float_as_uint(most) + 0x1fffffu) >> 23;   // one more where the significand is over 1.75
  return exponent > 9 ? exponent - 8 : 1;
}

// 2^e of a scale byte, and its reciprocal for a byte from scale_byte (1 to 247).
__device__ inline float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ inline float inverse_scale_of(uint32_t byte) { return __uint_as_float((254 - byte) << 23); }

__device__ inline float magnitude(float x) { return fabsf(x) < __builtin_inff() ? fabsf(x) : 0.0f; }

// Four values as codes.
__device__ inline uint32_t code_word(float a, float b, float c, float d, float inverse) {
  auto scaled = [&](float x) { return fabsf(x) < __builtin_inff() ? x * inverse : __builtin_nanf(""); };
  int word = __builtin_amdgcn_cvt_pk_fp8_f32(scaled(a), scaled(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(scaled(c), scaled(d), word, true);
}

// What four codes stand for, but for the scale.
__device__ inline float4 decode_word(uint32_t word) {
  const f32x2 low = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false), high = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
  return make_float4(low.x, low.y, high.x, high.y);
}

// One row by one wave: elements `from`, `from` + stride, .. of `rows` to code words and the scale byte.  Whether what this lane
// holds of it is finite.
__device__ inline bool store_row(const View &rows, uint64_t from, uint64_t stride, uint32_t words, uint32_t *codes,
                                 uint8_t *scale) {
  const uint32_t lane = threadIdx.x & 63;
  float4 held[kWordsHeld];
  float most = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kWordsHeld; ++i) {
    const uint32_t word = lane + 64 * i;
    if (word >= words) continue;
    const uint64_t at = from + 4 * word * stride;
    held[i] = make_float4(load_float_at(rows, at), load_float_at(rows, at + stride), load_float_at(rows, at + 2 * stride),
                          load_float_at(rows, at + 3 * stride));
    most = fmaxf(fmaxf(fmaxf(most, magnitude(held[i].x)), fmaxf(magnitude(held[i].y), magnitude(held[i].z))),
                 magnitude(held[i].w));
  }
  const uint32_t byte = scale_byte(wave_max(most));
#pragma unroll
  for (uint32_t i = 0; i < kWordsHeld; ++i) {
    const uint32_t word = lane + 64 * i;
    if (word < words)
      codes[word] = code_word(held[i].x, held[i].y, held[i].z, held[i].w, inverse_scale_of(byte));
  }
  if (lane == 0) *scale = (uint8_t)byte;
  bool finite = true;
#pragma unroll
  for (uint32_t i = 0; i < kWordsHeld; ++i)
    if (lane + 64 * i < words)
      finite = finite && fabsf(held[i].x) < __builtin_inff() && fabsf(held[i].y) < __builtin_inff() &&
               fabsf(held[i].z) < __builtin_inff() && fabsf(held[i].w) < __builtin_inff();
  return finite;
}

// A row by `kLanes` lanes of a wave, eight values each: rows whose values lie together, in pieces of 16 bytes.
bool in_pieces(const View &rows, uint32_t width) {
  return rows.stride[2] == 1 && rows.stride[0] % 8 == 0 && rows.stride[1] % 8 == 0 && rows.offset % 8 == 0 && width % 8 == 0;
}

template <int kPattern>
__device__ inline float max_with(float x) {   // of lanes that a data-parallel pattern pairs
  const int other = __builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), kPattern, 0xf, 0xf, true);
  return fmaxf(x, __uint_as_float((uint32_t)other));
}

template <uint32_t kLanes>
__device__ inline float max_of_lanes(float x) {
  x = max_with<0xb1>(x);    // lane ^ 1
  x = max_with<0x4e>(x);    // lane ^ 2
  x = max_with<0x141>(x);   // the other four of eight
  if constexpr (kLanes >= 16) x = max_with<0x140>(x);   // the other eight of sixteen
  if constexpr (kLanes >= 32) {
    const auto v = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
  }
  return x;
}

struct Piece {
  float x[8];
};

// Eight values as they are in memory.
struct RawPiece {
  uint4 words[2];   // [1]: of f32 alone
};

__device__ inline RawPiece load_raw(const void *rows, uint32_t dtype, uint64_t from) {
  RawPiece v;
  if (dtype == FH_F32) {
    v.words[0] = *(const uint4 *)((const float *)rows + from);
    v.words[1] = *(const uint4 *)((const float *)rows + from + 4);
  } else {
    v.words[0] = *(const uint4 *)((const uint16_t *)rows + from);
  }
  return v;
}

__device__ inline Piece values_of(const RawPiece &raw, uint32_t dtype) {
  const uint32_t words[8] = {raw.words[0].x, raw.words[0].y, raw.words[0].z, raw.words[0].w,
                             raw.words[1].x, raw.words[1].y, raw.words[1].z, raw.words[1].w};
  Piece v;
  if (dtype == FH_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v.x[i] = __uint_as_float(words[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v.x[2 * i] = dtype == FH_F16 ? f16_to_f32((uint16_t)words[i]) : bf16_to_f32((uint16_t)words[i]);
      v.x[2 * i + 1] = dtype == FH_F16 ? f16_to_f32((uint16_t)(words[i] >> 16)) : bf16_to_f32((uint16_t)(words[i] >> 16));
    }
  }
  return v;
}

// This lane's eight values (of the row's piece `piece`) to codes, lane 0 of the row the scale byte.  Whether they are finite.
template <uint32_t kLanes>
__device__ inline bool store_piece(const Piece &v, uint32_t piece, uint8_t *codes, uint8_t *scale) {
  float most = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    most = fmaxf(most, magnitude(v.x[i]));
    finite = finite && fabsf(v.x[i]) < __builtin_inff();
  }
  const uint32_t byte = scale_byte(max_of_lanes<kLanes>(most));
  const float inverse = inverse_scale_of(byte);
  *(uint2 *)(codes + 8 * piece) = make_uint2(code_word(v.x[0], v.x[1], v.x[2], v.x[3], inverse), code_word(v.x[4], v.x[5], v.x[6], v.x[7], inverse));
  if (piece == 0) *scale = (uint8_t)byte;
  return finite;
}

// Where a row's codes (in words) and scale (in bytes) are.
__device__ inline uint64_t code_at(const View &codes, uint64_t page, uint32_t slot, uint32_t head, uint32_t page_tokens,
                                   uint32_t heads, uint32_t words) {
  return codes.offset + ((page * page_tokens + slot) * heads + head) * words;
}

// ---- one sequence: rows into its pages and out of them ----

__device__ inline bool quant_page(const QuantCopy &p, uint64_t position, ErrorSlot *error, bool reports, uint32_t *page) {
  const uint64_t logical = position / p.page_tokens;
  const uint32_t *table = (const uint32_t *)p.table.base + p.table.offset;
  const uint32_t *generations = (const uint32_t *)p.generations.base + p.generations.offset;
  if (entry_ok(table, generations, (uint32_t)logical, p.logical_pages, p.physical_pages, page)) return true;
  if (reports) report_error(error, (uint32_t)logical);
  return false;
}

__device__ inline bool quant_active(const View &activity) {
  return !activity.base || ((const uint32_t *)activity.base)[activity.offset] != 0;
}

// A wave per row.
__global__ __launch_bounds__(256) void quant_store_kernel(QuantCopy p, ErrorSlot *error) {
  const uint64_t row = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (uint64_t)p.tokens * p.heads || !quant_active(p.activity)) return;
  const uint32_t token = (uint32_t)(row / p.heads), head = (uint32_t)(row % p.heads);
  const uint64_t position = (uint64_t)p.start + token;
  uint32_t page;
  if (!quant_page(p, position, error, (threadIdx.x & 63) == 0, &page)) return;
  const uint32_t slot = (uint32_t)(position % p.page_tokens);
  store_row(p.rows, p.rows.offset + token * p.rows.stride[0] + head * p.rows.stride[1], p.rows.stride[2], p.words,
            (uint32_t *)p.codes.base + code_at(p.codes, page, slot, head, p.page_tokens, p.heads, p.words),
            (uint8_t *)p.scales.base + 4 * (p.scales.offset + page * p.scales.stride[0] + head * p.scale_words) + slot);
}

// The same in pieces.  What bounds it: the vector ALUs, which find row, head, page and slot for every eight values (177 instructions a
// wave, busy 0.75 of the time), next to HBM; of few rows the chain table, generation, store.  (32749 rows of 8 heads of 128, 101 MB:
// 27 us, 3.7 TB/s; by the kernel above 105.)
template <uint32_t kLanes>
__global__ __launch_bounds__(256) void quant_store_rows_kernel(QuantCopy p, ErrorSlot *error) {
  const uint32_t flat = blockIdx.x * 256 + threadIdx.x, row = flat / kLanes, piece = flat % kLanes;
  if (row >= p.tokens * p.heads || !quant_active(p.activity)) return;
  const uint32_t token = row / p.heads, head = row - token * p.heads;
  const RawPiece raw = load_raw(p.rows.base, p.rows.dtype, p.rows.offset + token * p.rows.stride[0] + head * p.rows.stride[1] + 8 * piece);
  const uint64_t position = (uint64_t)p.start + token;
  uint32_t page;
  if (!quant_page(p, position, error, piece == 0, &page)) return;   // (all lanes of a row)
  const uint32_t slot = (uint32_t)(position % p.page_tokens);
  store_piece<kLanes>(values_of(raw, p.rows.dtype), piece, (uint8_t *)((uint32_t *)p.codes.base + code_at(p.codes, page, slot, head, p.page_tokens, p.heads, p.words)),
                      (uint8_t *)p.scales.base + 4 * (p.scales.offset + page * p.scales.stride[0] + head * p.scale_words) + slot);
}

// Eight codes a thread out of the pages.  What bounds it: the chain table, generation, codes, store of every wave (waiting 0.61 of its
// time), two rounds of workgroups of it for 16384 rows of 4 heads of 128 to f32 (42 MB: 13.5 us, 3.1 TB/s; the kernel below 18).
__global__ __launch_bounds__(256) void quant_load_rows_kernel(QuantCopy p, ErrorSlot *error) {
  const uint32_t flat = blockIdx.x * 256 + threadIdx.x, pieces = p.words / 2;
  if (flat >= p.tokens * p.heads * pieces || !quant_active(p.activity)) return;
  const uint32_t row = flat / pieces, piece = flat - row * pieces, token = row / p.heads, head = row - token * p.heads;
  const uint64_t position = (uint64_t)p.start + token;
  uint32_t page;
  if (!quant_page(p, position, error, piece == 0, &page)) return;
  const uint32_t slot = (uint32_t)(position % p.page_tokens);
  const uint2 codes =
      *(const uint2 *)((const uint32_t *)p.codes.base + code_at(p.codes, page, slot, head, p.page_tokens, p.heads, p.words) + 2 * piece);
  const float scale = scale_of(
      ((const uint8_t *)p.scales.base)[4 * (p.scales.offset + page * p.scales.stride[0] + head * p.scale_words) + slot]);
  const float4 low = decode_word(codes.x), high = decode_word(codes.y);
  const float x[8] = {low.x * scale, low.y * scale, low.z * scale, low.w * scale, high.x * scale, high.y * scale, high.z * scale, high.w * scale};
  const uint64_t at = p.rows.offset + token * p.rows.stride[0] + head * p.rows.stride[1] + 8 * piece;
  if (p.rows.dtype == FH_F32) {
    *(float4 *)((float *)p.rows.base + at) = make_float4(x[0], x[1], x[2], x[3]);
    *(float4 *)((float *)p.rows.base + at + 4) = make_float4(x[4], x[5], x[6], x[7]);
    return;
  }
  uint32_t words[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    words[i] = p.rows.dtype == FH_F16 ? f32_to_f16(x[2 * i]) | (uint32_t)f32_to_f16(x[2 * i + 1]) << 16
                                      : f32_to_bf16(x[2 * i]) | (uint32_t)f32_to_bf16(x[2 * i + 1]) << 16;
  *(uint4 *)((uint16_t *)p.rows.base + at) = make_uint4(words[0], words[1], words[2], words[3]);
}

// A thread per code word.
__global__ __launch_bounds__(256) void quant_load_kernel(QuantCopy p, ErrorSlot *error) {
  const uint64_t flat = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (flat >= (uint64_t)p.tokens * p.heads * p.words || !quant_active(p.activity)) return;
  const uint32_t word = (uint32_t)(flat % p.words), head = (uint32_t)(flat / p.words % p.heads);
  const uint32_t token = (uint32_t)(flat / p.words / p.heads);
  const uint64_t position = (uint64_t)p.start + token;
  uint32_t page;
  if (!quant_page(p, position, error, word == 0, &page)) return;
  const uint32_t slot = (uint32_t)(position % p.page_tokens);
  const float4 value = decode_word(
      ((const uint32_t *)p.codes.base)[code_at(p.codes, page, slot, head, p.page_tokens, p.heads, p.words) + word]);
  const float scale = scale_of(
      ((const uint8_t *)p.scales.base)[4 * (p.scales.offset + page * p.scales.stride[0] + head * p.scale_words) + slot]);
  const uint64_t at = p.rows.offset + token * p.rows.stride[0] + head * p.rows.stride[1] + 4 * word * p.rows.stride[2];
  store_float_at(p.rows, at, value.x * scale);
  store_float_at(p.rows, at + p.rows.stride[2], value.y * scale);
  store_float_at(p.rows, at + 2 * p.rows.stride[2], value.z * scale);
  store_float_at(p.rows, at + 3 * p.rows.stride[2], value.w * scale);
}

// ---- a packed ragged batch ----

__global__ __launch_bounds__(256) void quant_validate_kernel(const uint32_t *cu, uint32_t lanes, uint32_t tokens,
                                                             uint32_t *flag, ErrorSlot *error) {
  __shared__ uint32_t lowest;
  if (threadIdx.x == 0) lowest = 0xffffffffu;
  __syncthreads();
  const uint32_t mine = first_malformed_lane(cu, lanes, tokens, threadIdx.x, 256);
  if (mine != 0xffffffffu) atomicMin(&lowest, mine);
  __syncthreads();
  if (threadIdx.x == 0) {
    flag[0] = lowest != 0xffffffffu;
    if (lowest != 0xffffffffu) report_error(error, lowest);
  }
}

__device__ inline uint64_t scale_at(const RaggedQuantAttention &p, uint64_t page, uint32_t plane, uint32_t head) {
  return 4 * (p.scales.offset + ((page * 2 + plane) * p.kv_heads + head) * p.scale_words);
}

// Stores every lane's new rows: a wave per (token, plane, head).
// (`mark`, unless null, gets `tag` if a value is not finite, and marks[token] too)
__global__ __launch_bounds__(256) void quant_append_kernel(RaggedQuantAttention p, ErrorSlot *error, const uint32_t *malformed,
                                                           uint32_t *mark, uint32_t *marks, uint32_t tag) {
  if (malformed[0]) return;
  const uint64_t row = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (uint64_t)p.tokens * 2 * p.kv_heads) return;
  const uint32_t token = (uint32_t)(row / (2 * p.kv_heads)), of = (uint32_t)(row % (2 * p.kv_heads));
  const uint32_t plane = of / p.kv_heads, head = of % p.kv_heads;
  const bool reports = of == 0 && (threadIdx.x & 63) == 0;
  const uint32_t *cu = (const uint32_t *)p.cu_seqlens.base + p.cu_seqlens.offset;
  if (token < cu[0] || token >= cu[p.lanes]) return;
  const uint32_t lane = find_lane(cu, p.lanes, token);
  if (p.one_row_per_lane && cu[lane + 1] - cu[lane] > 1) {   // the promise is broken: nothing of the lane is stored
    if (reports) report_error(error, token);
    return;
  }
  if (p.activity.base && ((const uint32_t *)p.activity.base)[p.activity.offset + lane] == 0) return;
  const uint64_t position = (uint64_t)((const uint32_t *)p.q_starts.base)[p.q_starts.offset + lane] + (token - cu[lane]);
  const uint64_t logical = position / p.page_tokens;
  const uint32_t *table = (const uint32_t *)p.tables.base + p.tables.offset + (uint64_t)lane * p.table_pages * 2;
  const uint32_t *generations = (const uint32_t *)p.generations.base + p.generations.offset;
  uint32_t page;
  if (logical >= p.table_pages || !entry_ok(table, generations, (uint32_t)logical, p.table_pages, p.physical_pages, &page)) {
    if (reports) report_error(error, logical > 0xffffffffull ? 0xffffffffu : (uint32_t)logical);
    return;
  }
  const View &rows = plane ? p.v_new : p.k_new, &codes = plane ? p.value_codes : p.key_codes;
  const uint32_t words = (plane ? p.value_width : p.width) / 4, slot = (uint32_t)(position % p.page_tokens);
  const bool finite = store_row(rows, rows.offset + token * rows.stride[0] + head * rows.stride[1], rows.stride[2], words,
                                (uint32_t *)codes.base + code_at(codes, page, slot, head, p.page_tokens, p.kv_heads, words),
                                (uint8_t *)p.scales.base + scale_at(p, page, plane, head) + slot);
  if (mark && plane && !finite) *mark = marks[token] = tag;
}

// Any width: one wave per (token, query head); a lane attends every 64th key with a softmax of its own, and the 64
// states are merged at the end.
template <int kMaxWords>
__global__ __launch_bounds__(64) void quant_attention_generic_kernel(RaggedQuantAttention p, ErrorSlot *error,
                                                                     const uint32_t *malformed) {
  __shared__ float4 q_row[128];
  __shared__ int bad;
  const uint32_t token = blockIdx.x / p.query_heads, head = blockIdx.x % p.query_heads, thread = threadIdx.x;
  const uint32_t *cu = (const uint32_t *)p.cu_seqlens.base + p.cu_seqlens.offset;
  const uint64_t out_base = p.out.offset + token * p.out.stride[0] + head * p.out.stride[1];
  const bool covered = !malformed[0] && token >= cu[0] && token < cu[p.lanes];
  const uint32_t lane = covered ? find_lane(cu, p.lanes, token) : 0;
  const bool active = covered && !(p.one_row_per_lane && cu[lane + 1] - cu[lane] > 1) &&
                      !(p.activity.base && ((const uint32_t *)p.activity.base)[p.activity.offset + lane] == 0);
  auto zero_row = [&] {
    for (uint32_t c = thread; c < p.value_width; c += 64) store_float_at(p.out, out_base + c * p.out.stride[2], 0.0f);
  };
  if (!active) return zero_row();
  const uint64_t attended =
      (uint64_t)((const uint32_t *)p.q_starts.base)[p.q_starts.offset + lane] + (token - cu[lane]) + 1;
  const uint32_t *table = (const uint32_t *)p.tables.base + p.tables.offset + (uint64_t)lane * p.table_pages * 2;
  const uint32_t *generations = (const uint32_t *)p.generations.base + p.generations.offset;
  if (thread == 0) bad = 0;
  __syncthreads();
  uint64_t pages = (attended + p.page_tokens - 1) / p.page_tokens;
  if (pages > p.table_pages) {
    if (thread == 0) {
      report_error(error, p.table_pages);
      bad = 1;
    }
    pages = p.table_pages;
  }
  for (uint32_t page = thread; page < pages; page += 64) {
    uint32_t physical;
    if (!entry_ok(table, generations, page, p.table_pages, p.physical_pages, &physical)) {
      report_error(error, page);
      bad = 1;
    }
  }
  const uint32_t key_words = p.width / 4, value_words = p.value_width / 4;
  for (uint32_t word = thread; word < key_words; word += 64) {
    const uint64_t at = p.q.offset + token * p.q.stride[0] + head * p.q.stride[1] + 4 * word * p.q.stride[2];
    q_row[word] = make_float4(load_float_at(p.q, at), load_float_at(p.q, at + p.q.stride[2]),
                              load_float_at(p.q, at + 2 * p.q.stride[2]), load_float_at(p.q, at + 3 * p.q.stride[2]));
  }
  __syncthreads();
  if (bad) return zero_row();
  const uint32_t kv_head = head / (p.query_heads / p.kv_heads);
  float m = -__builtin_inff(), l = 0.0f;
  float4 acc[kMaxWords];
#pragma unroll
  for (int c = 0; c < kMaxWords; ++c) acc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (uint64_t key = thread; key < attended; key += 64) {
    const uint32_t page = table[2 * (key / p.page_tokens)], slot = (uint32_t)(key % p.page_tokens);
    const uint32_t *k = (const uint32_t *)p.key_codes.base + code_at(p.key_codes, page, slot, kv_head, p.page_tokens, p.kv_heads, key_words);
    const uint32_t *v = (const uint32_t *)p.value_codes.base + code_at(p.value_codes, page, slot, kv_head, p.page_tokens, p.kv_heads, value_words);
    const float k_scale = scale_of(((const uint8_t *)p.scales.base)[scale_at(p, page, 0, kv_head) + slot]);
    const float v_scale = scale_of(((const uint8_t *)p.scales.base)[scale_at(p, page, 1, kv_head) + slot]);
    float score = 0.0f;
    for (uint32_t word = 0; word < key_words; ++word) {
      const float4 x = decode_word(k[word]), y = q_row[word];
      score += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
    }
    score *= k_scale * p.scale;
    const float m_new = fmaxf(m, score);
    const float correction = m == -__builtin_inff() ? 0.0f : expf(m - m_new);
    const float w = score == -__builtin_inff() ? 0.0f : expf(score - m_new);   // (a state may have met nothing else yet)
    l = l * correction + w;
#pragma unroll
    for (int c = 0; c < kMaxWords; ++c)
      if ((uint32_t)c < value_words) {
        const float4 x = decode_word(v[c]);
        const float weight = w * v_scale;
        acc[c].x = acc[c].x * correction + weight * x.x;
        acc[c].y = acc[c].y * correction + weight * x.y;
        acc[c].z = acc[c].z * correction + weight * x.z;
        acc[c].w = acc[c].w * correction + weight * x.w;
      }
    m = m_new;
  }
  const float m_all = wave_max(m);
  const float factor = m == -__builtin_inff() ? 0.0f : expf(m - m_all);
  const float l_all = wave_sum(l * factor);
#pragma unroll
  for (int c = 0; c < kMaxWords; ++c) {
    if ((uint32_t)c >= value_words) continue;
    const float4 sum = make_float4(wave_sum(acc[c].x * factor), wave_sum(acc[c].y * factor), wave_sum(acc[c].z * factor),
                                   wave_sum(acc[c].w * factor));
    if (thread == 0) {
      const uint64_t at = out_base + 4 * c * p.out.stride[2];
      store_float_at(p.out, at, sum.x / l_all);
      store_float_at(p.out, at + p.out.stride[2], sum.y / l_all);
      store_float_at(p.out, at + 2 * p.out.stride[2], sum.z / l_all);
      store_float_at(p.out, at + 3 * p.out.stride[2], sum.w / l_all);
    }
  }
}

// ---- the fast form: bf16, f16 or f32 queries, heads of 64 or 128 values, pages of whole 16 tokens ----
//
// A work plan (one launch, shared by the layers of a submission) cuts every lane's rows into units and their keys
// into splits; the splits are attended, and the units of several merged.  (The kernels above on the same batches: one lane of
// 400 keys 63 us instead of 8, 8 f32 lanes of 256 to 32768 keys 1750 instead of 20, 512 f32 prompt rows 496 instead of 25.)

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

constexpr uint32_t kTile = 32;            // keys of a step of the decode kernel
// Of the merge kernel.  One token of 30011 keys in up to 256 splits 11.4 + 5.7 us, in up to 128 14.9 + 5.0; tokens of up to 4
// splits by a quarter-row of threads 4.9 us (128 lanes), of up to 8 6.2.
constexpr uint32_t kMergeThreads = 256, kMostSplits = kMergeThreads, kFewSplits = 4;
// Of the prompt kernel; kPromptGrid: its workgroups a compute unit, of which two run at once (2048 rows and 32 lanes 92 us, with
// two in all 103: who ends early finds nothing more).
constexpr uint32_t kPromptWaves = 4, kPromptRows = 32 * kPromptWaves, kPromptTile = 64, kPromptGrid = 8;
constexpr uint32_t kPlanLanes = 4096;     // lanes that the plan holds
// Keys of a split at least, where a decode batch fits the device at once: 400 keys in splits of 64 7.7 us, of 128 10.4; their
// merge is no slower.
constexpr uint32_t kLeastSplit = 64;
// And of one token's beside units of several: 32 lanes beside 2048 prompt rows 92 us, from 512 up to 4096 96 (beside 64
// prompt rows 25.6 and 24.2).
constexpr uint32_t kMixedLeast = 256, kMixedMost = 1024;
// Units of several tokens: each split of theirs costs members x heads partial rows, written and read (a row's split about as much
// as attending 300 keys).  They are split where the device has places to spare, into at least the first many keys (512 rows of one
// prompt: 25 us and 5 of merge; into 128 keys 26 and 6.6); and into the second where places would be left empty behind the
// first round.
constexpr uint32_t kPromptLeast = 256, kPromptSplit = 4096;

// One split of a unit: `members` consecutive tokens of a lane from `leader` on, the first of which attends `attended` keys.
// The partial results of member m and split s go to slot base + m * (its kind's most splits) + s.
struct alignas(16) QuantItem {
  uint32_t leader, split, lane, attended;
  uint32_t chunk, splits, members, base;
};

struct QuantBatch {
  const void *q, *k_new, *v_new;   // of q_dtype; strides below count their elements
  void *out;                       // of out_dtype
  uint8_t *key_codes, *value_codes, *scales;
  const uint32_t *tables, *generations, *cu, *starts, *activity;
  uint64_t q_stride_t, q_stride_h, out_stride_t, out_stride_h, kn_stride_t, kn_stride_h, vn_stride_t, vn_stride_h;
  uint32_t q_dtype, out_dtype;
  uint32_t tokens, lanes, query_heads, kv_heads, group, head_tiles;   // head_tiles: of up to 16 query heads to a kv head
  uint32_t page_tokens, scale_bytes, physical_pages, table_pages;     // scale_bytes: of a head's tokens in a page
  // Tokens of a unit of a lane that brings several; 0: every token is a unit of its own (a decode batch).
  uint32_t prompt_tokens;
  uint32_t max_splits, prompt_splits;   // most splits of a unit of one token and of others
  uint32_t single_slots;                // partial slots of units of one token, in front of those of others
  uint32_t item_slots;                  // workgroups that the device holds at once, over those of an item of one token
  uint32_t promised, append_in_kernel;
  uint32_t not_finite;                  // what counts[4] holds if a new value row is not finite, and not_finite_rows of its token
  float scale_log2;
  // work plan
  uint32_t *bad;            // [T] a page of the token was refused
  uint4 *merge;             // [T] what the merge writes: token, splits, first partial slot; from the front tokens of many splits, from
                            // the back those of few and zero rows (no split)
  uint2 *tokens_of;         // [T] a token's lane, and the keys it attends (0: of no lane, or past its table)
  QuantItem *items;         // units of several tokens first
  uint32_t *counts;         // [0] items, [1] entries of `merge` from the front, [2] non-zero: cu_seqlens was refused, [3] items of
                            // several tokens, [4] see not_finite, [5] entries of `merge` from the back
  uint32_t *not_finite_rows;   // [T]
  float *partial_o;         // [slots, Hq, D]
  float2 *partial_ml;       // [slots, Hq]
};

// Splits of a unit of `keys` keys: as few as keep each within `split_keys`, of equal length in whole tiles.
__device__ inline void split_unit(uint32_t keys, uint32_t split_keys, uint32_t max_splits, uint32_t *chunk, uint32_t *splits) {
  const uint32_t want = min((keys - 1) / split_keys + 1, max_splits);
  const uint32_t even = (keys + want - 1) / want;
  *chunk = (even + kTile - 1) / kTile * kTile;
  *splits = (keys + *chunk - 1) / *chunk;
}

// Of a token's new rows (keys, then values) those from `begin` to `end` by one wave: what is the token's (lane, position, page)
// is found once, the first piece of every lane on its way meanwhile.  What bounds it: the chain of start, table entry,
// generation and store; of many rows HBM.  (A thread to a piece, finding the page for itself, is bound by that arithmetic: 8256
// rows of 8 heads 19 us.  More pieces of a lane on their way take room from waves: four 18 us, one 15.8.)
template <uint32_t kLanes>
__device__ inline void store_new_rows(const QuantBatch &p, ErrorSlot *error, uint32_t token, uint32_t begin, uint32_t end, uint32_t lane,
                                      uint64_t position) {
  constexpr uint32_t kRows = 64 / kLanes;
  const uint32_t heads = 2 * p.kv_heads, thread = threadIdx.x & 63, piece = thread % kLanes, first = begin + thread / kLanes;
  auto request = [&](uint32_t of) {
    return of >= p.kv_heads ? load_raw(p.v_new, p.q_dtype, token * p.vn_stride_t + (of - p.kv_heads) * p.vn_stride_h + 8 * piece)
                            : load_raw(p.k_new, p.q_dtype, token * p.kn_stride_t + of * p.kn_stride_h + 8 * piece);
  };
  RawPiece raw;
  if (first < end) raw = request(first);
  const uint64_t logical = position / p.page_tokens;
  const uint32_t slot = (uint32_t)(position - logical * p.page_tokens);
  uint32_t page;
  if (logical >= p.table_pages ||
      !entry_ok(p.tables + (uint64_t)lane * p.table_pages * 2, p.generations, (uint32_t)logical, p.table_pages, p.physical_pages, &page)) {
    if (thread == 0) report_error(error, logical > 0xffffffffull ? 0xffffffffu : (uint32_t)logical);
    return;
  }
  const uint64_t row0 = ((uint64_t)page * p.page_tokens + slot) * p.kv_heads;
  uint8_t *scales = p.scales + (uint64_t)page * heads * p.scale_bytes + slot;
  for (uint32_t of = first; of < end; of += kRows) {   // (all lanes of a row)
    if (of != first) raw = request(of);
    const bool value = of >= p.kv_heads;
    uint8_t *codes = value ? p.value_codes + (row0 + of - p.kv_heads) * (8 * kLanes) : p.key_codes + (row0 + of) * (8 * kLanes);
    if (!store_piece<kLanes>(values_of(raw, p.q_dtype), piece, codes, scales + (uint64_t)of * p.scale_bytes) && value)
      p.counts[4] = p.not_finite_rows[token] = p.not_finite;
  }
}

// Stores the new rows of a batch whose plan is made: a wave for a token's keys, and one for its values (one for both: 8256
// tokens 15.8 us instead of 14.3).
template <uint32_t kLanes>
__global__ __launch_bounds__(256) void quant_append_rows_kernel(QuantBatch p, ErrorSlot *error) {
  const uint32_t token = __builtin_amdgcn_readfirstlane(blockIdx.x * 2 + (threadIdx.x >> 7));
  if (token >= p.tokens) return;
  const uint32_t begin = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6 & 1) * p.kv_heads;
  const uint2 planned = p.tokens_of[token];
  if (planned.y != 0) store_new_rows<kLanes>(p, error, token, begin, begin + p.kv_heads, planned.x, planned.y - 1);
}

// `op` over the sixteen lanes of a row, and over the wave: every lane gets the result.
template <typename Op>
__device__ inline uint32_t row_reduce(uint32_t x, Op op) {
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true));
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, true));
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true));
  return op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, true));
}
template <typename Op>
__device__ inline uint32_t wave_reduce(uint32_t x, Op op) {
  x = row_reduce(x, op);
  const auto rows = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = op(rows[0], rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return op(halves[0], halves[1]);
}

// What the workgroups of a work plan hold in LDS.
template <uint32_t kThreads>
struct PlanShared {
  static constexpr uint32_t kLanes = kThreads == 1024 ? kPlanLanes : kThreads;
  static constexpr uint32_t kWaves = kThreads / 64, kUnitsHeld = 2 * kThreads, kClasses = 128, kTrials = 16;
  uint32_t lane_cu[kLanes + 1], lane_start[kLanes], unit_first[kLanes + 1];
  uint32_t unit_tiles[kUnitsHeld], class_items[kClasses], wave_sums[kWaves], trial[kTrials];
  uint16_t unit_lane[kUnitsHeld];
  uint32_t total_tiles, prompt_tiles;   // of 32 keys
  uint32_t malformed, longest, prompt_longest, prompt_units, merge_count, few_count, units, idle_lanes;
};

// By one workgroup.  What bounds it: dependent steps, every one a memory round trip or a barrier.
template <uint32_t kThreads>
__device__ inline void make_plan(const QuantBatch &p, PlanShared<kThreads> &s, ErrorSlot *error) {
  using S = PlanShared<kThreads>;
  const uint32_t thread = threadIdx.x, lane_id = thread & 63, wave = thread >> 6;
  for (uint32_t l = thread; l < p.lanes; l += kThreads) {
    s.lane_start[l] = p.starts[l];
    s.unit_first[l] = !p.activity || p.activity[l] != 0;   // whether it is active, until its units are counted
  }
  for (uint32_t c = thread; c < S::kClasses; c += kThreads) s.class_items[c] = 0;
  if (thread == 0) {
    s.total_tiles = s.prompt_tiles = 0;
    s.longest = s.prompt_longest = s.prompt_units = s.merge_count = s.few_count = s.idle_lanes = 0;
  }
  __syncthreads();
  // A refused cu_seqlens fails the whole dispatch: zero rows, nothing stored, the lowest offending lane reported.
  if (s.malformed != 0xffffffffu) {
    for (uint32_t token = thread; token < p.tokens; token += kThreads) {
      p.tokens_of[token] = make_uint2(0, 0);
      p.merge[token] = make_uint4(token, 0, 0, 0);
    }
    if (thread == 0) {
      report_error(error, s.malformed);
      p.counts[0] = p.counts[3] = 0;
      p.counts[1] = 0;
      p.counts[5] = p.tokens;
      p.counts[2] = 1;
    }
    return;
  }
  // Units of this thread's lanes, and of those before them.
  const uint32_t per_thread = (p.lanes + kThreads - 1) / kThreads, lane0 = min(thread * per_thread, p.lanes),
                 lane1 = min(lane0 + per_thread, p.lanes);
  auto unit_tokens = [&](uint32_t n) { return p.prompt_tokens == 0 || n == 1 ? 1 : p.prompt_tokens; };
  auto units_of = [&](uint32_t n) { return p.promised && n > 1 ? 0u : (n + unit_tokens(n) - 1) / unit_tokens(n); };
  uint32_t mine = 0;
  for (uint32_t l = lane0; l < lane1; ++l) mine += s.unit_first[l] ? units_of(s.lane_cu[l + 1] - s.lane_cu[l]) : 0;
  uint32_t sum = mine;
  for (int offset = 1; offset < 64; offset <<= 1) {
    const uint32_t before = __shfl_up(sum, offset, 64);
    if ((int)lane_id >= offset) sum += before;
  }
  if (lane_id == 63) s.wave_sums[wave] = sum;
  __syncthreads();
  uint32_t at = sum - mine;
  for (uint32_t w = 0; w < wave; ++w) at += s.wave_sums[w];
  // A zero row: entry `place` of the list from the back.
  auto zero_row = [&](uint32_t token, uint32_t place) {
    p.tokens_of[token] = make_uint2(0, 0);
    p.merge[p.tokens - 1 - place] = make_uint4(token, 0, 0, 0);
  };
  for (uint32_t l = lane0; l < lane1; ++l) {
    const uint32_t first = s.lane_cu[l], last = s.lane_cu[l + 1], active = s.unit_first[l], own = active ? units_of(last - first) : 0;
    s.unit_first[l] = at;
    for (uint32_t unit = at; unit < min(at + own, S::kUnitsHeld); ++unit) s.unit_lane[unit] = (uint16_t)l;
    at += own;
    if (own == 0 && first < last) {
      if (active) report_error(error, first);   // the caller's promise does not hold
      s.idle_lanes = 1;
    }
  }
  if (thread == kThreads - 1) s.unit_first[p.lanes] = s.units = at;
  // Rows of no lane come first in the list of zero rows, then those of lanes without units, a wave to a lane.  (By one thread
  // each: 10 rows padded to 8192 took 362 us in all, now 41.)
  const uint32_t covered = s.lane_cu[0], behind = s.lane_cu[p.lanes];
  for (uint32_t token = thread; token < covered; token += kThreads) zero_row(token, token);
  for (uint32_t token = behind + thread; token < p.tokens; token += kThreads) zero_row(token, covered + (token - behind));
  if (thread == 0) s.few_count = covered + (p.tokens - behind);
  __syncthreads();
  const uint32_t units = s.units;
  if (s.idle_lanes)
    for (uint32_t l = wave; l < p.lanes; l += S::kWaves) {
      const uint32_t first = s.lane_cu[l], rows = s.unit_first[l + 1] == s.unit_first[l] ? s.lane_cu[l + 1] - first : 0;
      if (rows == 0) continue;
      uint32_t place = lane_id == 0 ? atomicAdd(&s.few_count, rows) : 0;
      place = __builtin_amdgcn_readfirstlane(place);
      for (uint32_t i = lane_id; i < rows; i += 64) zero_row(first + i, place + i);
    }
  const uint64_t most_keys = min((uint64_t)p.table_pages * p.page_tokens, (uint64_t)0xffffffffu);
  // A unit's lane, first token, tokens, and keys of the last of them (0: none); and the tokens behind them that pass the lane's table.
  struct Unit {
    uint32_t lane, token, members, keys, past;
    bool prompt;   // of a lane that brings several tokens
  };
  auto unit_at = [&](uint32_t unit) {
    Unit u;
    u.lane = unit < S::kUnitsHeld ? s.unit_lane[unit] : find_lane(s.unit_first, p.lanes, unit);
    const uint32_t n = s.lane_cu[u.lane + 1] - s.lane_cu[u.lane], each = unit_tokens(n), index = (unit - s.unit_first[u.lane]) * each;
    u.prompt = p.prompt_tokens != 0 && n > 1;
    u.token = s.lane_cu[u.lane] + index;
    const uint32_t all = min(each, n - index);
    const uint64_t before = (uint64_t)s.lane_start[u.lane] + index;
    u.members = before < most_keys ? (uint32_t)min((uint64_t)all, most_keys - before) : 0u;
    u.past = all - u.members;
    u.keys = u.members ? (uint32_t)before + u.members : 0u;
    return u;
  };
  {
    uint32_t tiles_sum = 0, prompt_sum = 0, tiles_longest = 0, prompt_long = 0, prompts = 0;
    for (uint32_t unit = thread; unit < units; unit += kThreads) {
      const Unit u = unit_at(unit);
      const uint32_t tiles = (u.keys + kTile - 1) / kTile;
      if (unit < S::kUnitsHeld) s.unit_tiles[unit] = tiles;
      if (u.prompt) {
        prompt_sum += tiles;
        prompt_long = max(prompt_long, tiles);
        ++prompts;
      } else {
        tiles_sum += tiles;
        tiles_longest = max(tiles_longest, tiles);
      }
    }
    tiles_sum = wave_reduce(tiles_sum, [](uint32_t x, uint32_t y) { return x + y; });
    tiles_longest = wave_reduce(tiles_longest, [](uint32_t x, uint32_t y) { return max(x, y); });
    if (lane_id == 0 && tiles_sum) {
      atomicAdd(&s.total_tiles, tiles_sum);
      atomicMax(&s.longest, tiles_longest);
    }
    if (p.prompt_tokens != 0) {
      prompt_sum = wave_reduce(prompt_sum, [](uint32_t x, uint32_t y) { return x + y; });
      prompts = wave_reduce(prompts, [](uint32_t x, uint32_t y) { return x + y; });
      prompt_long = wave_reduce(prompt_long, [](uint32_t x, uint32_t y) { return max(x, y); });
      if (lane_id == 0 && prompts) {
        atomicAdd(&s.prompt_tiles, prompt_sum);
        atomicAdd(&s.prompt_units, prompts);
        atomicMax(&s.prompt_longest, prompt_long);
      }
    }
  }
  __syncthreads();
  uint32_t split_keys, prompt_split = 0;
  if (p.prompt_tokens != 0) {
    // A quarter of what a place has to do in all, so that the splits of one token's keys, started last, level its end.
    const uint32_t share = (uint32_t)(((uint64_t)s.prompt_tiles * p.kv_heads + s.total_tiles) / (4 * p.item_slots));
    split_keys = min(max(min(share, kMixedMost / kTile) * kTile, kMixedLeast), kMixedMost);
    // entries of the launch's list, against the workgroups that the device holds
    const uint32_t entries = max(s.prompt_units * p.kv_heads, 1u), held = p.item_slots * ((p.kv_heads * p.head_tiles + kPromptWaves - 1) / kPromptWaves);
    const uint32_t parts = held / entries, rounds = (4 * held + entries - 1) / entries;
    if (parts >= 2)
      prompt_split = max((s.prompt_longest + parts - 1) / parts * kTile, kPromptLeast);
    else if (entries > held && rounds > 1)
      prompt_split = max((s.prompt_longest + rounds - 1) / rounds * kTile, kPromptSplit);
    else
      prompt_split = 0xffffffffu / 2;
  } else {
    // The shortest split length whose items all find a place on the device at once: one item per place costs each place one
    // start-up and leaves no second, partly filled round behind.  Between the even share of a place and twice it, by sixteenths,
    // sixteen threads to a length; where none does (the units alone outnumber the places, or nearly), the even share.
    const uint32_t even = max((s.total_tiles + p.item_slots - 1) / p.item_slots, kLeastSplit / kTile);
    auto length = [&](uint32_t trial) { return even + (even * trial + S::kTrials - 1) / S::kTrials; };   // in tiles
    uint32_t first = 0;
    if (units * p.max_splits > p.item_slots) {
      for (uint32_t trial = thread / 16; trial < S::kTrials; trial += kThreads / 16) {
        const float inverse = 1.0f / (float)length(trial);
        uint32_t items = 0;
        for (uint32_t unit = thread % 16; unit < units; unit += 16) {
          const uint32_t tiles = unit < S::kUnitsHeld ? s.unit_tiles[unit] : (unit_at(unit).keys + kTile - 1) / kTile;
          items += min((uint32_t)ceilf((float)tiles * inverse - 1e-3f), p.max_splits);
        }
        items = row_reduce(items, [](uint32_t x, uint32_t y) { return x + y; });
        if (thread % 16 == 0) s.trial[trial] = items <= p.item_slots;
      }
      __syncthreads();
      while (first < S::kTrials && !s.trial[first]) ++first;
    }
    split_keys = (first < S::kTrials ? length(first) : even) * kTile;
  }
  // Units of several tokens first, and by length, longest first, so that the launch, which starts items in list order, ends
  // on its shortest.
  auto split_of = [&](const Unit &u, uint32_t *chunk, uint32_t *splits) {
    split_unit(u.keys, u.prompt ? prompt_split : split_keys, u.prompt ? p.prompt_splits : p.max_splits, chunk, splits);
    return (u.prompt ? 64 : 0) + min(*chunk / kTile, 63u);
  };
  auto base_of = [&](const Unit &u) {
    return u.prompt ? p.single_slots + u.token * p.prompt_splits : (p.prompt_tokens ? u.lane : u.token) * p.max_splits;
  };
  // Eight threads a unit, for its tokens and splits; one where the units are many and each is a token.
  const uint32_t each = p.prompt_tokens != 0 || 8 * units <= kThreads ? 8 : 1, part = thread % each;
  for (uint32_t unit = thread / each; unit < units; unit += kThreads / each) {
    const Unit u = unit_at(unit);
    uint32_t chunk = 0, splits = 1, listed = 0;
    if (u.keys != 0) {
      const uint32_t of = split_of(u, &chunk, &splits);
      if (part == 0) atomicAdd(&s.class_items[of], splits);
    }
    if (part == 0 && splits != 1) listed = atomicAdd(splits > kFewSplits ? &s.merge_count : &s.few_count, u.members);
    listed = __shfl(listed, (int)(lane_id - part), 64);
    const uint32_t base = base_of(u);
    for (uint32_t m = part; m < u.members; m += each) {
      p.bad[u.token + m] = 0;
      p.tokens_of[u.token + m] = make_uint2(u.lane, u.keys - u.members + m + 1);
      if (splits != 1) p.merge[splits > kFewSplits ? listed + m : p.tokens - 1 - listed - m] = make_uint4(u.token + m, splits, base + m * p.prompt_splits, 0);
    }
    if (part == 0 && u.past != 0) {
      report_error(error, p.table_pages);
      const uint32_t first = u.token + u.members, place = atomicAdd(&s.few_count, u.past);
      for (uint32_t m = 0; m < u.past; ++m) zero_row(first + m, place + m);
    }
  }
  __syncthreads();
  if (wave == 0) {   // class counts -> first item of each class
    uint32_t running = 0;
    for (int first = S::kClasses - 1; first >= 0; first -= 64) {
      const uint32_t count = s.class_items[first - lane_id];
      uint32_t before = count;
      for (int offset = 1; offset < 64; offset <<= 1) {
        const uint32_t other = __shfl_up(before, offset, 64);
        if ((int)lane_id >= offset) before += other;
      }
      s.class_items[first - lane_id] = running + before - count;
      running += __shfl(before, 63, 64);
      if (lane_id == 0 && first == S::kClasses - 1) p.counts[3] = running;
    }
    if (lane_id == 0) {
      p.counts[0] = running;
      p.counts[1] = s.merge_count;
      p.counts[5] = s.few_count;
      p.counts[2] = 0;
    }
  }
  __syncthreads();
  for (uint32_t unit = thread / each; unit < units; unit += kThreads / each) {
    const Unit u = unit_at(unit);
    if (u.keys == 0) continue;
    uint32_t chunk, splits, first = 0;
    const uint32_t of = split_of(u, &chunk, &splits);
    if (part == 0) first = atomicAdd(&s.class_items[of], splits);
    first = __shfl(first, (int)(lane_id - part), 64);
    for (uint32_t split = part; split < splits; split += each)
      p.items[first + split] = QuantItem{u.token, split, u.lane, u.keys - u.members + 1, chunk, splits, u.members, base_of(u)};
  }
}

// One launch for what stands in front of a submission's first attention: workgroup 0 makes the plan, the others store the
// batch's new rows meanwhile, a wave a token (none where the rows do not come in pieces of 16 bytes).
template <uint32_t kThreads, uint32_t kLanes>
__global__ __launch_bounds__(kThreads) void quant_prepare_kernel(QuantBatch p, ErrorSlot *error) {
  __shared__ PlanShared<kThreads> s;
  if (threadIdx.x == 0) s.malformed = 0xffffffffu;
  for (uint32_t l = threadIdx.x; l <= p.lanes; l += kThreads) s.lane_cu[l] = p.cu[l];
  __syncthreads();
  for (uint32_t l = threadIdx.x; l < p.lanes; l += kThreads)
    if (s.lane_cu[l + 1] < s.lane_cu[l] || s.lane_cu[l + 1] > p.tokens) atomicMin(&s.malformed, l);
  __syncthreads();
  if (blockIdx.x == 0) return make_plan<kThreads>(p, s, error);
  if (s.malformed != 0xffffffffu) return;
  for (uint32_t i = (blockIdx.x - 1) * (kThreads / 64) + (threadIdx.x >> 6); i < p.tokens; i += (gridDim.x - 1) * (kThreads / 64)) {
    const uint32_t token = __builtin_amdgcn_readfirstlane(i);
    if (token < s.lane_cu[0] || token >= s.lane_cu[p.lanes]) continue;
    const uint32_t lane = __builtin_amdgcn_readfirstlane(find_lane(s.lane_cu, p.lanes, token));
    const uint32_t first = __builtin_amdgcn_readfirstlane(s.lane_cu[lane]), last = __builtin_amdgcn_readfirstlane(s.lane_cu[lane + 1]);
    if ((p.promised && last - first > 1) || (p.activity && p.activity[lane] == 0)) continue;
    store_new_rows<kLanes>(p, error, token, 0, 2 * p.kv_heads, lane, (uint64_t)p.starts[lane] + (token - first));
  }
}

__device__ inline uint32_t pack_bf16(float lo, float hi) {
  const bf16x2 v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ inline uint32_t pack_f16(float lo, float hi) {
  const f16x2 v = {(_Float16)lo, (_Float16)hi};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ inline float low_bf16(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ inline float high_bf16(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// The larger of a value's two lanes (l, l + 32), and of its four (l, l + 16, ..).
__device__ inline float max_of_halves(float x) {
  const auto v = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
}
__device__ inline float max_of_quarters(float x) {
  const auto v = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max_of_halves(fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1])));
}

// 16 consecutive query elements as they are in memory (kWide false: bf16), and as f32.
template <bool kWide>
struct RawQuery {
  uint4 words[kWide ? 4 : 2];   // f32 alone has four
};

template <bool kWide>
__device__ inline void request_query(const QuantBatch &p, uint64_t element, RawQuery<kWide> &raw) {
  if (kWide && p.q_dtype == FH_F32) {
#pragma unroll
    for (int i = 0; i < (kWide ? 4 : 2); ++i) raw.words[i] = *(const uint4 *)((const float *)p.q + element + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) raw.words[i] = *(const uint4 *)((const uint16_t *)p.q + element + 8 * i);
  }
}

template <bool kWide>
__device__ inline void query_values(const QuantBatch &p, const RawQuery<kWide> &raw, float (&x)[16]) {
  if (kWide && p.q_dtype == FH_F32) {
#pragma unroll
    for (int i = 0; i < (kWide ? 4 : 2); ++i) {
      x[4 * i] = __uint_as_float(raw.words[i].x), x[4 * i + 1] = __uint_as_float(raw.words[i].y);
      x[4 * i + 2] = __uint_as_float(raw.words[i].z), x[4 * i + 3] = __uint_as_float(raw.words[i].w);
    }
    return;
  }
  const uint32_t w[8] = {raw.words[0].x, raw.words[0].y, raw.words[0].z, raw.words[0].w,
                         raw.words[1].x, raw.words[1].y, raw.words[1].z, raw.words[1].w};
  if (kWide && p.q_dtype == FH_F16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f16x2 pair = __builtin_bit_cast(f16x2, w[i]);
      x[2 * i] = (float)pair.x;
      x[2 * i + 1] = (float)pair.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[2 * i] = low_bf16(w[i]);
      x[2 * i + 1] = high_bf16(w[i]);
    }
  }
}

// The queries of a wave's 16 rows (this lane: 16 elements of each 64, of row `lane & 15`) as operands of the matrix cores.
//   kWide false: e4m3 pieces x = 2^e (c_0 + c_1 / 16) for the scaled products with the codes as they are.  Two hold the 8
//     bits of a bf16 element down to 2^-11 of the row's largest, and what is smaller to 2^-22 of it.  (These products sum terms
//     of any size to 2^-14 of the largest, root mean square, at worst to 2^-11 of it or 2^-12 of the sum of all sizes; a large
//     term beside small ones to 2^-16, at worst 2^-12.7; operands within a factor of nine exactly.  For scores of a few units
//     that is below what bf16 weights round.)
//   kWide true: f16 pieces x = 2^e (h_0 + h_1 / 2^11), 22 bits, for products with the codes as f16.
template <int D, bool kWide>
struct Queries {
  uint32_t piece[2][D / 64][kWide ? 8 : 4];
  uint32_t exponent;   // the byte of 2^e
};

// The byte of a row's 2^e.  The second e4m3 pieces count 2^(e - 4), whose byte has to be one too: 5 at least (rows below 2^-113;
// their elements then lie lower in the codes' range, and the smallest come to 2^-135, far below what their scores tell apart).
template <bool kWide>
__device__ inline uint32_t query_scale_byte(float most) {
  const uint32_t byte = scale_byte(most);
  return kWide ? byte : max(byte, 5u);
}

// Sixteen query elements as pieces; `inverse`: 2^-e.  (No number stays one: its code, or f16's.)
template <bool kWide>
__device__ inline void query_pieces(const float (&x)[16], float inverse, uint32_t *first, uint32_t *second) {
  if constexpr (kWide) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = x[2 * i] * inverse, b = x[2 * i + 1] * inverse;
      first[i] = pack_f16(a, b);
      const f16x2 held = __builtin_bit_cast(f16x2, first[i]);
      second[i] = pack_f16((a - (float)held.x) * 2048.0f, (b - (float)held.y) * 2048.0f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = x[4 * i + j] * inverse;
      int word = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      word = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], word, true);
      const float4 held = decode_word((uint32_t)word);
      first[i] = (uint32_t)word;
      auto rest = [](float value, float part) { return __builtin_fmaf(part, -16.0f, value * 16.0f); };
      word = __builtin_amdgcn_cvt_pk_fp8_f32(rest(y[0], held.x), rest(y[1], held.y), 0, false);
      second[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(rest(y[2], held.z), rest(y[3], held.w), word, true);
    }
  }
}

// An infinite element makes its row's scores no numbers, as the no number it becomes here does.
template <int N>
__device__ inline float largest_query(float (&x)[N][16]) {
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(x[j][i]));
  if (__any(most == __builtin_inff())) {
    most = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (fabsf(x[j][i]) == __builtin_inff()) x[j][i] = __builtin_nanf("");
        most = fmaxf(most, fabsf(x[j][i]));
      }
  }
  return most;
}

// (the rows' elements have been requested: `raw`)
template <int D, bool kWide>
__device__ inline void make_queries(const QuantBatch &p, Queries<D, kWide> &q, const RawQuery<kWide> (&raw)[D / 64], bool used) {
  float x[D / 64][16];
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    query_values<kWide>(p, raw[j], x[j]);
    if (!used)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[j][i] = 0.0f;
  }
  q.exponent = query_scale_byte<kWide>(max_of_quarters(largest_query(x)));
#pragma unroll
  for (int j = 0; j < D / 64; ++j) query_pieces<kWide>(x[j], inverse_scale_of(q.exponent), q.piece[0][j], q.piece[1][j]);
}

// One tile of 32 keys in registers.  Lane (t = lane & 15, g = lane >> 4) holds 16 of each 64 elements of key t of either
// half, and of the 8 keys 4g .. 4g + 3 of either half the D / 16 value columns from (D / 16) t on.
template <int D>
struct QuantTile {
  static constexpr int kColumns = D / 16, kWords = kColumns / 4;
  uint32_t k[2][D / 64][4];
  uint32_t v[8][kWords];
  uint32_t k_scale[2], v_scale[2];   // four tokens' bytes; k_scale of the narrow form: the byte of key t
};

struct LaneOffsets {
  uint32_t k, v;       // bytes from the first row of a half
  uint32_t row_bytes;  // of a token's rows of all heads
};

template <int D, bool kWide>
__device__ inline void load_tile(const QuantBatch &p, QuantTile<D> &r, uint32_t tile0, uint32_t end, uint32_t page0,
                                 uint32_t physical, const LaneOffsets &at, uint32_t kv_head, uint32_t t, uint32_t g) {
  const uint32_t pt = p.page_tokens;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    // A half never straddles a page: it is a buffer of its rows up to `end`.  What lies past a buffer's length reads as
    // zeros and is not fetched (unused slots may hold anything, and 0 * NaN would poison the sums).
    const uint32_t first = tile0 + 16 * half, rows = end > first ? min(end - first, 16u) : 0;
    const uint32_t token = min(first, (end - 1) & ~15u);   // a half past the end has no rows: any page will do
    const uint32_t page = __builtin_amdgcn_readlane(physical, __builtin_amdgcn_readfirstlane(token / pt - page0));
    const uint32_t slot = __builtin_amdgcn_readfirstlane(token % pt);
    const uint64_t row0 = ((uint64_t)page * pt + slot) * at.row_bytes;
    const int bytes = __builtin_amdgcn_readfirstlane(rows * at.row_bytes);
    const auto k_rows = __builtin_amdgcn_make_buffer_rsrc((void *)(p.key_codes + row0), 0, bytes, 0x27000);
    const auto v_rows = __builtin_amdgcn_make_buffer_rsrc((void *)(p.value_codes + row0), 0, bytes, 0x27000);
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(k_rows, (int)(at.k + 64 * j), 0, 2 /* streamed */);
      r.k[half][j][0] = v.x, r.k[half][j][1] = v.y, r.k[half][j][2] = v.z, r.k[half][j][3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int from = (int)(at.v + i * at.row_bytes);
      if constexpr (D == 64) {
        r.v[4 * half + i][0] = __builtin_amdgcn_raw_buffer_load_b32(v_rows, from, 0, 2);
      } else {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(v_rows, from, 0, 2);
        r.v[4 * half + i][0] = v.x, r.v[4 * half + i][1] = v.y;
      }
    }
    // (a page's scales are whole: what lies past `end` is masked where it is used)
    const uint8_t *scales = p.scales + ((uint64_t)page * 2 * p.kv_heads + kv_head) * p.scale_bytes + slot;
    if constexpr (kWide)
      r.k_scale[half] = *(const uint32_t *)(scales + 4 * g);
    else
      r.k_scale[half] = scales[t];
    r.v_scale[half] = *(const uint32_t *)(scales + (uint64_t)p.kv_heads * p.scale_bytes + 4 * g);
  }
}

struct Softmax {
  float m, l;
};

// 2^e of byte j of four.
__device__ inline float scale_in(uint32_t word, int j) {
  return __uint_as_float((j < 3 ? word << (23 - 8 * j) : word >> 1) & 0x7f800000u);
}

// Scores, online softmax and the value product for one tile against 16 query rows (this lane holds row t).  `limit`: the
// first key that may not be attended; kMasked false: none of the tile's.
template <int D, bool kWide, bool kMasked>
__device__ inline void consume_tile(const QuantTile<D> &cur, const Queries<D, kWide> &q, f32x4 (&o)[D / 16], Softmax &sm,
                                    uint32_t tile0, uint32_t limit, float scale_log2, uint32_t g) {
  float s_val[8];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if constexpr (kWide) {
      f32x4 low = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < D / 64; ++j)
#pragma unroll
        for (int part = 0; part < 2; ++part) {   // 8 of the lane's 16 elements
          uint32_t a[4];
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            a[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(cur.k[half][j][2 * part + w], 1.0f, false));
            a[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(cur.k[half][j][2 * part + w], 1.0f, true));
          }
          const f16x8 keys = __builtin_bit_cast(f16x8, make_uint4(a[0], a[1], a[2], a[3]));
          auto piece = [&](int i) {
            const uint32_t *w = q.piece[i][j] + 4 * part;
            return __builtin_bit_cast(f16x8, make_uint4(w[0], w[1], w[2], w[3]));
          };
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, piece(0), acc, 0, 0, 0);
          low = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, piece(1), low, 0, 0, 0);
        }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        s_val[4 * half + j] = __builtin_amdgcn_ldexpf(__builtin_fmaf(low[j], 1.0f / 2048.0f, acc[j]),
                                                      (int)((cur.k_scale[half] >> 8 * j & 0xff) + q.exponent) - 254) * scale_log2;
    } else {
#pragma unroll
      for (int i = 1; i >= 0; --i)
#pragma unroll
        for (int j = 0; j < D; j += 128) {
          i32x8 a, b;
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            a[w] = D == 64 && w >= 4 ? 0 : (int)cur.k[half][D == 64 ? 0 : j / 64 + w / 4][w & 3];
            b[w] = D == 64 && w >= 4 ? 0 : (int)q.piece[i][D == 64 ? 0 : j / 64 + w / 4][w & 3];
          }
          acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 0, (int)cur.k_scale[half], 0, (int)(q.exponent - 4 * i));
        }
#pragma unroll
      for (int j = 0; j < 4; ++j) s_val[4 * half + j] = acc[j] * scale_log2;
    }
  }
  if constexpr (kMasked)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (tile0 + 16 * (i >> 2) + 4 * g + (i & 3) >= limit) s_val[i] = -__builtin_inff();
  float tile_max = s_val[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) tile_max = fmaxf(tile_max, s_val[i]);
  tile_max = max_of_quarters(tile_max);
  const float m_new = fmaxf(sm.m, tile_max);
  // a row that has met nothing but -inf yet keeps m = -inf; subtract 0 instead so that exp2(-inf) = 0
  const float m_safe = m_new == -__builtin_inff() ? 0.0f : m_new;
  float w_val[8], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float weight = __builtin_amdgcn_exp2f(s_val[i] - m_safe);
    sum += weight;
    w_val[i] = weight * scale_in(cur.v_scale[i >> 2], i & 3);
    if (kMasked && tile0 + 16 * (i >> 2) + 4 * g + (i & 3) >= limit) w_val[i] = 0.0f;
  }
  // The running maximum settles after a few tiles; skip the rescale when no lane's moved.
  if (__any(m_new != sm.m)) {
    const float alpha = __builtin_amdgcn_exp2f(sm.m - m_safe);   // 0 while m is -inf
    sm.l *= alpha;
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[mt][j] *= alpha;
    sm.m = m_new;
  }
  sm.l += sum;
  // The weights: two bf16 each (16 bits; with one the errors of bf16 rows against 64 bits are 0.0019 instead of 0.0017, most of it
  // the output's rounding, and no batch is faster), or three that hold all their 24 bits.
  constexpr int kPieces = kWide ? 3 : 2;
  uint32_t pieces[kPieces][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = w_val[2 * i], y = w_val[2 * i + 1];
#pragma unroll
    for (int piece = 0; piece < kPieces; ++piece) {
      pieces[piece][i] = pack_bf16(x, y);
      x -= low_bf16(pieces[piece][i]);
      y -= high_bf16(pieces[piece][i]);
    }
  }
  // O^T += V^T . P^T, four columns of the lane's at a time: two keys' codes of a column side by side make a pair.
#pragma unroll
  for (int word = 0; word < QuantTile<D>::kWords; ++word) {
    uint32_t pairs[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pairs[i][0] = __builtin_amdgcn_perm(cur.v[2 * i + 1][word], cur.v[2 * i][word], 0x05010400u);
      pairs[i][1] = __builtin_amdgcn_perm(cur.v[2 * i + 1][word], cur.v[2 * i][word], 0x07030602u);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        a[i] = __builtin_bit_cast(uint32_t, c & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(pairs[i][c >> 1], 1.0f, true)
                                                  : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(pairs[i][c >> 1], 1.0f, false));
      const bf16x8 values = __builtin_bit_cast(bf16x8, make_uint4(a[0], a[1], a[2], a[3]));
      const int mt = 4 * word + c;
#pragma unroll
      for (int piece = kPieces - 1; piece >= 0; --piece)
        o[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            values, __builtin_bit_cast(bf16x8, make_uint4(pieces[piece][0], pieces[piece][1], pieces[piece][2], pieces[piece][3])),
            o[mt], 0, 0, 0);
    }
  }
}

// Four consecutive output elements from `element` on.
__device__ inline void store_out4(const QuantBatch &p, uint64_t element, float a, float b, float c, float d) {
  if (p.out_dtype == FH_F32)
    *(float4 *)((float *)p.out + element) = make_float4(a, b, c, d);
  else if (p.out_dtype == FH_F16)
    *(uint2 *)((uint16_t *)p.out + element) = make_uint2(pack_f16(a, b), pack_f16(c, d));
  else
    *(uint2 *)((uint16_t *)p.out + element) = make_uint2(pack_bf16(a, b), pack_bf16(c, d));
}

// One new row of D values by one wave: codes and the scale byte.
template <int D>
__device__ inline void append_row(const void *rows, uint32_t dtype, uint64_t from, uint8_t *codes, uint8_t *scale) {
  constexpr int kEach = D / 64;
  const uint32_t lane = threadIdx.x & 63;
  float x[kEach], most = 0.0f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const uint64_t at = from + kEach * lane + i;
    x[i] = dtype == FH_F32 ? ((const float *)rows)[at]
                           : (dtype == FH_F16 ? f16_to_f32(((const uint16_t *)rows)[at]) : bf16_to_f32(((const uint16_t *)rows)[at]));
    most = fmaxf(most, magnitude(x[i]));
  }
  const uint32_t byte = scale_byte(wave_max(most));
  const uint32_t word = code_word(x[0], x[kEach - 1], 0.0f, 0.0f, inverse_scale_of(byte));
  if constexpr (kEach == 1)
    codes[lane] = (uint8_t)word;
  else
    ((uint16_t *)codes)[lane] = (uint16_t)word;
  if (lane == 0) *scale = (uint8_t)byte;
}

// One split of a unit of one token, for up to 16 query heads of one kv head, by one wave.
template <int D, bool kWide>
__device__ inline void attend_token(const QuantBatch &p, ErrorSlot *error, const QuantItem &item, uint32_t kv_head, uint32_t head_tile) {
  uint32_t lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));   // what follows from it is not kept in registers from item to item
  const uint32_t t = lane & 15, g = lane >> 4, pt = p.page_tokens;
  const uint32_t begin = item.split * item.chunk, end = min(item.attended, begin + item.chunk);
  const uint32_t *table = p.tables + (uint64_t)item.lane * p.table_pages * 2;
  const uint32_t first_page = begin / pt, last_page = (end - 1) / pt;
  // What does not wait for anything is requested first: up to 64 table entries at once, and the queries.
  auto request_entry = [&](uint32_t page0) {
    return page0 + lane <= last_page ? *(const uint2 *)(table + 2 * (uint64_t)(page0 + lane)) : make_uint2(0, 0);
  };
  uint2 entry = request_entry(first_page);
  const uint32_t head = kv_head * p.group + 16 * head_tile + t;
  const bool used = 16 * head_tile + t < p.group;
  RawQuery<kWide> raw[D / 64];   // (an unused row takes the first's)
#pragma unroll
  for (int j = 0; j < D / 64; ++j)
    request_query<kWide>(p, item.leader * p.q_stride_t + (used ? head : kv_head * p.group) * p.q_stride_h + 64 * j + 16 * g, raw[j]);
  if (p.append_in_kernel && item.split + 1 == item.splits) {
    // This wave's kv head of the lane's new rows goes into the cache before anything is read: the rows sit at the last
    // attended position, which only the last split's range contains.
    const uint32_t position = item.attended - 1;
    uint32_t page;
    if (entry_ok(table, p.generations, position / pt, p.table_pages, p.physical_pages, &page)) {
      const uint32_t slot = position % pt;
      const uint64_t row = (((uint64_t)page * pt + slot) * p.kv_heads + kv_head) * D;
      uint8_t *scale = p.scales + ((uint64_t)page * 2 * p.kv_heads + kv_head) * p.scale_bytes + slot;
      append_row<D>(p.k_new, p.q_dtype, item.leader * p.kn_stride_t + kv_head * p.kn_stride_h, p.key_codes + row, scale);
      append_row<D>(p.v_new, p.q_dtype, item.leader * p.vn_stride_t + kv_head * p.vn_stride_h, p.value_codes + row,
                    scale + (uint64_t)p.kv_heads * p.scale_bytes);
      __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): the loads below come from the same wave, after the stores
    }   // else: the page walk below meets the same entry and ends the item
  }
  Queries<D, kWide> q;
  LaneOffsets at;
  at.row_bytes = p.kv_heads * D;
  at.k = t * at.row_bytes + kv_head * D + 16 * g;
  at.v = 4 * g * at.row_bytes + kv_head * D + D / 16 * t;
  f32x4 o[D / 16];
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt) o[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  Softmax sm{-__builtin_inff(), 0.0f};
  // The first tile of 64 pages is requested beside their generations: a page that is there may be read, and what a refused one
  // holds is not used.
  QuantTile<D> a, b;
  uint32_t physical, generation, low, high;
  auto open_pages = [&](uint32_t page0) {
    physical = entry.x < p.physical_pages ? entry.x : 0;
    generation = p.generations[physical];
    low = max(begin, page0 * pt);
    high = (uint32_t)min((uint64_t)end, ((uint64_t)page0 + 64) * pt);
    load_tile<D, kWide>(p, a, low, high, page0, physical, at, kv_head, t, g);
  };
  open_pages(first_page);
  make_queries<D, kWide>(p, q, raw, used);
  for (uint32_t page0 = first_page;;) {
    const unsigned long long bad_mask = __ballot(page0 + lane <= last_page && (physical != entry.x || generation != entry.y));
    if (bad_mask) {
      if (lane == (uint32_t)__ffsll((long long)bad_mask) - 1) {
        report_error(error, page0 + lane);
        p.bad[item.leader] = 1;
      }
      if (item.splits == 1 && used) {   // no merge follows
        const uint64_t row = item.leader * p.out_stride_t + head * p.out_stride_h;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) store_out4(p, row + D / 4 * g + 4 * c, 0.f, 0.f, 0.f, 0.f);
      }
      return;
    }
    // Two tiles in registers, in turns: one is requested while the other is on its way, and neither is moved (a move waits
    // for it, and with it for every load before).  Only the last may be partial.
    uint32_t tile0 = low, left = (high - low + kTile - 1) / kTile;
    for (; left > 2; left -= 2, tile0 += 2 * kTile) {
      load_tile<D, kWide>(p, b, tile0 + kTile, high, page0, physical, at, kv_head, t, g);
      __builtin_amdgcn_sched_barrier(0);
      consume_tile<D, kWide, false>(a, q, o, sm, tile0, high, p.scale_log2, g);
      __builtin_amdgcn_sched_barrier(0);
      load_tile<D, kWide>(p, a, tile0 + 2 * kTile, high, page0, physical, at, kv_head, t, g);
      __builtin_amdgcn_sched_barrier(0);
      consume_tile<D, kWide, false>(b, q, o, sm, tile0 + kTile, high, p.scale_log2, g);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (left == 2) {
      load_tile<D, kWide>(p, b, tile0 + kTile, high, page0, physical, at, kv_head, t, g);
      __builtin_amdgcn_sched_barrier(0);
      consume_tile<D, kWide, false>(a, q, o, sm, tile0, high, p.scale_log2, g);
      __builtin_amdgcn_sched_barrier(0);
      consume_tile<D, kWide, true>(b, q, o, sm, tile0 + kTile, high, p.scale_log2, g);
    } else {
      consume_tile<D, kWide, true>(a, q, o, sm, tile0, high, p.scale_log2, g);
    }
    if (page0 + 64 > last_page) break;
    page0 += 64;
    entry = request_entry(page0);
    open_pages(page0);
  }
  sm.l += __shfl_xor(sm.l, 16, 64);
  sm.l += __shfl_xor(sm.l, 32, 64);
  if (!used) return;
  // Lane (row t, group g) holds value columns D / 16 * (4g + j) + mt of its row in o[mt][j].
  const bool single = item.splits == 1;
  const float inverse = single ? 1.0f / sm.l : 1.0f;
  const uint64_t slot = (uint64_t)(item.base + item.split) * p.query_heads + head;
  const uint64_t row = item.leader * p.out_stride_t + head * p.out_stride_h;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint32_t column = D / 16 * (4 * g + j) + 4 * c;
      const float x = o[4 * c][j] * inverse, y = o[4 * c + 1][j] * inverse, z = o[4 * c + 2][j] * inverse, w = o[4 * c + 3][j] * inverse;
      if (single)
        store_out4(p, row + column, x, y, z, w);
      else
        *(float4 *)(p.partial_o + slot * D + column) = make_float4(x, y, z, w);
    }
  if (!single && g == 0) p.partial_ml[slot] = make_float2(sm.m, sm.l);
}

// A workgroup is one item; its waves take one kv head (and 16 of its query heads) each, so that the rows of all heads of
// a token are requested close together in time.  What bounds it: HBM (128 lanes of 256 to 32768 keys, 888 MB: 156 us, 5.7 TB/s);
// of few keys the chain item, table entry and generation, codes, and the launch (400 keys 8.0 us).  In between the start of
// every item, next to four to eight tiles of it (48 lanes of 128 to 4096 keys, 115 MB: 26 us; 8 f32 lanes of up to 32768, 55 MB: 20).
template <int D, bool kWide>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void quant_decode_kernel(QuantBatch p, ErrorSlot *error) {
  const uint32_t place = blockIdx.y * (blockDim.x >> 6) + (threadIdx.x >> 6);
  // (the first item comes with the count: there is room for as many as there are workgroups)
  QuantItem item = p.items[blockIdx.x];
  const uint32_t items = p.counts[0];
  asm volatile("" : "+s"(item.leader), "+s"(item.chunk));   // loaded here, not where it is used
  if (place >= p.kv_heads * p.head_tiles) return;
  const uint32_t kv_head = place / p.head_tiles, head_tile = place % p.head_tiles;
  for (uint32_t i = blockIdx.x; i < items;) {
    attend_token<D, kWide>(p, error, item, kv_head, head_tile);
    i += gridDim.x;
    if (i < items) item = p.items[i];
  }
}

// ---- prompts: key and value tiles staged in LDS and shared by the four waves of a workgroup ----
//
// An item of several tokens and a kv head: 128 query rows (token-major, the group's heads inside), 32 to a wave.  All waves
// walk the same keys in tiles of 64: the keys' codes are moved straight into LDS, where the scaled products (of 32 x 32,
// 64 elements a step) take them as they are; the values become bf16, their scale with them, between memory and LDS, once
// for the four waves.  A tile is on its way while the one before is attended; one barrier a tile.
//
// The 16-byte piece p of a key's row r sits in slot p ^ (r & 7) (64 values: p ^ (r >> 1 & 3)): eight rows read at one piece
// use all banks once.  Piece p of a value's row r sits in slot p ^ ((r & 3) << 2 | (r >> 2 & 3)) (64 values: p ^
// ((r >> 1 & 1) << 2 | (r >> 2 & 3))): the transposing read takes 4 rows x 4 pieces at once, which the first term spreads
// over the banks.  (Conflicts are counted all the same: 3.6e7 cycles for 2048 rows behind 16384 keys, about a tenth of the time of 256
// compute units; which of the accesses make them is not known.)  Keys past the end of a split are taken from a valid row and
// masked; values past it are zeros.
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((address_space(3))) s16x4 *LdsPiece;
typedef __attribute__((address_space(3))) u32x4 *LdsWords;
typedef __attribute__((address_space(3))) uint32_t *LdsWord;
typedef __attribute__((address_space(3))) uint8_t *LdsByte;

// A staged tile: key codes, values, the keys' scale bytes.  Tiles are named by their LDS address.
template <int D>
struct Staged {
  static constexpr uint32_t kKeyRow = D, kValueRow = 2 * D, kValues = kPromptTile * kKeyRow,
                            kScales = kValues + kPromptTile * kValueRow, kBytes = kScales + kPromptTile;
  static constexpr uint32_t kPieces = D / 16;               // of a row of codes
  static constexpr uint32_t kLoads = D / 64;                // 16-byte loads a lane for a wave's 16 rows
  static constexpr uint32_t kRowsEach = 16 / kLoads;        // rows of one of them
  __device__ static uint32_t key_slot(uint32_t row) { return D == 64 ? row >> 1 & 3 : row & 7; }
  __device__ static uint32_t value_slot(uint32_t row) { return (D == 64 ? (row >> 1 & 1) << 2 : (row & 3) << 2) | (row >> 2 & 3); }
};

// A wave's share of a tile on its way: the codes of its 16 rows of values, their scales, and a key's scale.
template <int D>
struct Arriving {
  u32x4 values[Staged<D>::kLoads];
  uint32_t scales[Staged<D>::kLoads], key_scale;
};

// Bit 7 of every byte that is a code of no number.
__device__ inline uint32_t no_numbers(uint32_t codes) { return ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Where a wave's next 16 rows are: index into the 64 pages held and token slot in that page.
struct StageCursor {
  uint32_t page, slot;
};

// Where a lane's pieces of a tile are, from the start of the tiles in LDS on: of its wave's 16 rows as they are staged, and
// as operands.
template <int D, bool kWide>
struct TilePlaces {
  uint32_t key_from, value_from;                 // in memory, from the wave's first row on (rows of the first load)
  uint32_t key_to, value_to[Staged<D>::kLoads][2];
  uint32_t scale_to;
  uint32_t keys[D / 32], values[D / 32][2], scales;
};

template <int D, bool kWide>
__device__ inline TilePlaces<D, kWide> tile_places(uint32_t tiles, uint32_t row_bytes, uint32_t wave, uint32_t lane) {
  using S = Staged<D>;
  TilePlaces<D, kWide> at;
  const uint32_t row0 = lane / S::kPieces, piece = lane % S::kPieces, half = lane >> 5;
  at.key_from = row0 * row_bytes + 16 * (piece ^ S::key_slot(row0));   // (the slot of row0 + 8 is row0's)
  at.value_from = row0 * row_bytes + 16 * piece;
  at.key_to = tiles + 16 * wave * S::kKeyRow;
#pragma unroll
  for (uint32_t j = 0; j < S::kLoads; ++j) {
    const uint32_t row = 16 * wave + S::kRowsEach * j + row0, slot = S::value_slot(row);
    at.value_to[j][0] = tiles + S::kValues + row * S::kValueRow + 16 * (2 * piece ^ slot);
    at.value_to[j][1] = tiles + S::kValues + row * S::kValueRow + 16 * ((2 * piece + 1) ^ slot);
  }
  at.scale_to = tiles + S::kScales + 16 * wave + lane;
  const uint32_t k_row = lane & 31, k_at = S::kKeyRow * k_row, k_slot = S::key_slot(k_row);
#pragma unroll
  for (uint32_t i = 0; i < D / 32; ++i)   // kWide: piece 2 i + half; else pieces 4 c + 2 half and the next of each 64 values c
    at.keys[i] = tiles + k_at + 16 * ((kWide ? 2 * i + half : 4 * (i / 2) + 2 * half + i % 2) ^ k_slot);
  const uint32_t v_row = 4 * half + ((lane & 15) >> 2);   // of the eight that a read transposes
#pragma unroll
  for (uint32_t c = 0; c < D / 32; ++c) {
    const uint32_t v_piece = 4 * c + 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i)
      at.values[c][i] = tiles + S::kValues + S::kValueRow * (v_row + 8 * i) + 8 * (lane & 1) + 16 * (v_piece ^ S::value_slot(v_row + 8 * i));
  }
  at.scales = tiles + S::kScales + (kWide ? 4 * half : lane & 31);
  return at;
}

// 64 lanes x 16 bytes, lane i's from `base` + its offset, straight into LDS (see load_to_lds_16_at).
__device__ inline void load_to_lds_16_from(const uint8_t *base, uint32_t offset, uint32_t lds_address) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(lds_address);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(at) : "memory");
}

// Requests this wave's 16 rows of the tile at `tile0`: keys into LDS (`buffer` bytes on), values into registers.
template <int D, bool kWide>
__device__ inline void request_tile(const QuantBatch &p, Arriving<D> &in, const TilePlaces<D, kWide> &to, uint32_t buffer, uint32_t tile0,
                                    uint32_t end, const StageCursor &at, uint32_t physical, uint32_t kv_head, uint32_t wave, uint32_t lane) {
  using S = Staged<D>;
  const uint32_t block = tile0 + 16 * wave, row_bytes = p.kv_heads * D;
  const uint32_t page = __builtin_amdgcn_readlane(physical, at.page);
  const uint64_t base = ((uint64_t)page * p.page_tokens + at.slot) * row_bytes + kv_head * D;
  const uint8_t *keys = p.key_codes + base, *values = p.value_codes + base;
  const uint8_t *key_scales = p.scales + ((uint64_t)page * 2 * p.kv_heads + kv_head) * p.scale_bytes + at.slot;
  const uint8_t *value_scales = key_scales + (uint64_t)p.kv_heads * p.scale_bytes;
  const uint32_t row0 = lane / S::kPieces;
  if (block + 16 <= end) {
#pragma unroll
    for (uint32_t j = 0; j < S::kLoads; ++j) {
      in.values[j] = *(const u32x4 *)(values + S::kRowsEach * j * row_bytes + to.value_from);
      in.scales[j] = value_scales[S::kRowsEach * j + row0];
    }
    in.key_scale = key_scales[lane & 15];
#pragma unroll
    for (uint32_t j = 0; j < S::kLoads; ++j)
      load_to_lds_16_from(keys + S::kRowsEach * j * row_bytes, to.key_from, to.key_to + buffer + S::kRowsEach * j * S::kKeyRow);
  } else {   // rows past the end are taken from a valid one
    const uint32_t last = block < end ? end - 1 - block : 0;   // (past the end: the cursor stayed behind)
#pragma unroll
    for (uint32_t j = 0; j < S::kLoads; ++j) {
      const uint32_t row = S::kRowsEach * j + row0, held = min(row, last), back = row0 * row_bytes;
      in.values[j] = *(const u32x4 *)(values + (held * row_bytes + (to.value_from - back)));
      in.scales[j] = value_scales[held];
    }
    in.key_scale = key_scales[min(lane & 15, last)];
#pragma unroll
    for (uint32_t j = 0; j < S::kLoads; ++j) {
      const uint32_t row = S::kRowsEach * j + row0, held = min(row, last), back = row0 * row_bytes;
      load_to_lds_16_from(keys, held * row_bytes + (to.key_from - back), to.key_to + buffer + S::kRowsEach * j * S::kKeyRow);
    }
  }
}

// Puts what has arrived into the tile.  Values of no number at keys from `clean_from` on become zeros (see attend_unit).
template <int D, bool kWide>
__device__ inline void settle_tile(const Arriving<D> &in, const TilePlaces<D, kWide> &to, uint32_t buffer, uint32_t tile0, uint32_t end,
                                   uint32_t clean_from, uint32_t wave, uint32_t lane) {
  using S = Staged<D>;
  const uint32_t row0 = 16 * wave + lane / S::kPieces;
#pragma unroll
  for (uint32_t j = 0; j < S::kLoads; ++j) {
    const uint32_t key = tile0 + S::kRowsEach * j + row0;
    u32x4 codes = in.values[j];
    if (tile0 + 16 * wave + 16 > min(end, clean_from)) {
      if (key >= end) codes = u32x4{0, 0, 0, 0};
      if (key >= clean_from)
#pragma unroll
        for (int w = 0; w < 4; ++w) codes[w] &= ~((no_numbers(codes[w]) >> 7) * 0xffu);
    }
    const float scale = scale_of(in.scales[j]);
    uint32_t pairs[8];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      pairs[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[w], scale, false));
      pairs[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[w], scale, true));
    }
    *(LdsWords)(to.value_to[j][0] + buffer) = u32x4{pairs[0], pairs[1], pairs[2], pairs[3]};
    *(LdsWords)(to.value_to[j][1] + buffer) = u32x4{pairs[4], pairs[5], pairs[6], pairs[7]};
  }
  if (lane < 16) *(LdsByte)(to.scale_to + buffer) = (uint8_t)in.key_scale;
}

// The queries of a wave's 32 rows as operands (see Queries): this lane holds the half `lane >> 5` of each 64 (kWide: 32)
// elements of row `lane & 31`.
template <int D, bool kWide>
struct PromptQueries {
  uint32_t piece[2][D / 64][kWide ? 16 : 8];
  uint32_t exponent;
};

// `sign`: the sign of the score's scale goes into the queries, a zero scale into their values (no number and an infinity
// become the no number that zero times they are): the largest product is then the largest score.
template <int D, bool kWide>
__device__ inline void make_prompt_queries(const QuantBatch &p, PromptQueries<D, kWide> &q, const RawQuery<kWide> (&raw)[D / 32], float sign) {
  float x[D / 32][16];
#pragma unroll
  for (int j = 0; j < D / 32; ++j) query_values<kWide>(p, raw[j], x[j]);
  if (sign != 1.0f)
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[j][i] *= sign;
  q.exponent = query_scale_byte<kWide>(max_of_halves(largest_query(x)));
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
    query_pieces<kWide>(x[j], inverse_scale_of(q.exponent), q.piece[0][j / 2] + (kWide ? 8 : 4) * (j % 2),
                        q.piece[1][j / 2] + (kWide ? 8 : 4) * (j % 2));
}

__device__ inline f32x16 mfma_bf16(const uint4 &a, const uint4 &b, const f32x16 &c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Scores, online softmax and the value product of the tile `buffer` bytes on for a wave's 32 query rows; this lane holds row
// (lane & 31) and, of each 8 keys, the four of its half.  `limit` is the first key the row may not attend (0: unused row);
// `masked` false: every key of the tile is below every limit.  scale_log2 is positive.
//
// The sums follow every new maximum, so that the weight of the largest score is exactly 1 (with sums that follow only what is
// 2^8 times larger: 2048 rows 94 us instead of 99, errors against 64 bits 2.3e-3 instead of 2.0e-3).  bf16 rows weigh with one
// bf16, summed as it is rounded (with two, errors are 1.7e-3, most of it the output's own rounding, but the products are what bounds this kernel:
// 2048 rows and 32 lanes 111 -> 129 us in all, 8256 rows 250 -> 293).
template <int D, bool kWide>
__device__ inline void attend_tile(const QuantBatch &p, const TilePlaces<D, kWide> &at, uint32_t buffer, const PromptQueries<D, kWide> &q,
                                   f32x16 (&o)[D / 32], Softmax &sm, bool masked, uint32_t tile0, uint32_t limit, float scale_log2,
                                   uint32_t lane) {
  using S = Staged<D>;
  const uint32_t half = lane >> 5;
  f32x16 s[2];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
    const uint32_t from = buffer + 32 * b * S::kKeyRow;
    if constexpr (kWide) {
      f32x16 low;
#pragma unroll
      for (int i = 0; i < 16; ++i) low[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const u32x4 codes = *(LdsWords)(at.keys[j] + from);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t a[4];
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            a[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[2 * part + w], 1.0f, false));
            a[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[2 * part + w], 1.0f, true));
          }
          const f16x8 keys = __builtin_bit_cast(f16x8, make_uint4(a[0], a[1], a[2], a[3]));
          auto piece = [&](int i) {
            const uint32_t *w = q.piece[i][j / 2] + 8 * (j % 2) + 4 * part;
            return __builtin_bit_cast(f16x8, make_uint4(w[0], w[1], w[2], w[3]));
          };
          s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(keys, piece(0), s[b], 0, 0, 0);
          low = __builtin_amdgcn_mfma_f32_32x32x16_f16(keys, piece(1), low, 0, 0, 0);
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint32_t bytes = *(LdsWord)(at.scales + buffer + 32 * b + 8 * n);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[b][4 * n + i] = __builtin_amdgcn_ldexpf(__builtin_fmaf(low[4 * n + i], 1.0f / 2048.0f, s[b][4 * n + i]),
                                                    (int)((bytes >> 8 * i & 0xff) + q.exponent) - 254);
      }
    } else {
      const int scale = *(LdsByte)(at.scales + buffer + 32 * b);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const u32x4 first = *(LdsWords)(at.keys[2 * c] + from), second = *(LdsWords)(at.keys[2 * c + 1] + from);
        i32x8 a, high, low;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          a[w] = (int)(w < 4 ? first[w] : second[w - 4]);
          high[w] = (int)q.piece[0][c][w];
          low[w] = (int)q.piece[1][c][w];
        }
        s[b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, low, s[b], 0, 0, 0, scale, 0, (int)(q.exponent - 4));
        s[b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, high, s[b], 0, 0, 0, scale, 0, (int)q.exponent);
      }
    }
  }
  auto read_values = [&](int step, int c) {
    const s16x4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPiece)(at.values[c][0] + (buffer + 16 * step * S::kValueRow)));
    const s16x4 high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPiece)(at.values[c][1] + (buffer + 16 * step * S::kValueRow)));
    const uint2 low_words = __builtin_bit_cast(uint2, low), high_words = __builtin_bit_cast(uint2, high);
    return make_uint4(low_words.x, low_words.y, high_words.x, high_words.y);
  };
  uint4 values[D / 32];   // operands one step ahead
#pragma unroll
  for (int c = 0; c < D / 32; ++c) values[c] = read_values(0, c);
  __builtin_amdgcn_sched_barrier(0);
  if (masked) {   // of the lane's keys 8 (i >> 2) + (i & 3) of block b, those below `below` are attended
    const uint32_t below = limit > tile0 + 4 * half ? limit - tile0 - 4 * half : 0;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (32 * b + 8 * (i >> 2) + (i & 3) >= below) s[b][i] = -__builtin_inff();
  }
  float largest = s[0][0];
#pragma unroll
  for (int i = 1; i < 32; ++i) largest = fmaxf(largest, s[i >> 4][i & 15]);
  largest = max_of_halves(largest) * scale_log2;
  if (__any(largest > sm.m)) {
    const float m_new = fmaxf(sm.m, largest), alpha = m_new == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(sm.m - m_new);
    sm.l *= alpha;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[c][i] *= alpha;
    sm.m = m_new;
  }
  // a row with nothing to attend yet keeps m = -inf; subtract 0 instead so that exp2(-inf) = 0
  const float m_safe = sm.m == -__builtin_inff() ? 0.0f : sm.m;
  constexpr int kPieces = kWide ? 3 : 1;
  // O^T += V^T . P^T, 16 keys a step in the order the scores left them: half h takes keys 4h..4h+3 and 8 + 4h..8 + 4h + 3 of
  // the 16.
#pragma unroll
  for (int step = 0; step < 4; ++step) {
    uint32_t words[kPieces][4];
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const int b = step >> 1, j = 8 * (step & 1) + i;
      float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][j], scale_log2, -m_safe));
      float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][j + 1], scale_log2, -m_safe));
      if constexpr (kWide) {
        sum[0] += x;
        sum[1] += y;
      }
#pragma unroll
      for (int piece = 0; piece < kPieces; ++piece) {
        words[piece][i / 2] = pack_bf16(x, y);
        x -= low_bf16(words[piece][i / 2]);
        y -= high_bf16(words[piece][i / 2]);
      }
      if constexpr (!kWide)
        sum[i >> 1 & 1] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, words[0][i / 2]), __builtin_bit_cast(bf16x2, 0x3f803f80u),
                                                          sum[i >> 1 & 1], false);
    }
    sm.l += sum[0] + sum[1];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
#pragma unroll
      for (int piece = kPieces - 1; piece >= 0; --piece)
        o[c] = mfma_bf16(values[c], make_uint4(words[piece][0], words[piece][1], words[piece][2], words[piece][3]), o[c]);
      if (step < 3) values[c] = read_values(step + 1, c);
    }
  }
}

// One item of several tokens for one kv head.
template <int D, bool kWide>
__device__ inline void attend_unit(const QuantBatch &p, ErrorSlot *error, uint32_t tiles, const QuantItem &item, uint32_t kv_head) {
  using S = Staged<D>;
  uint32_t lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));   // what follows from it is not kept in registers from item to item
  const uint32_t half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pt = p.page_tokens;
  const uint32_t longest = item.attended + item.members - 1;
  const uint32_t begin = item.split * item.chunk, end = min(longest, begin + item.chunk);
  const uint32_t *table = p.tables + (uint64_t)item.lane * p.table_pages * 2;
  const uint32_t first_page = begin / pt;
  uint32_t last_page = (end - 1) / pt;
  uint32_t refused_from = 0xffffffffu;   // the first key of the first page that is refused: rows that attend it are zeros
  // What does not wait for anything is requested first: up to 64 table entries at once (by every wave for itself: same
  // entries, same result), and the queries.
  auto request_entry = [&](uint32_t page0) {
    return page0 + lane <= last_page ? *(const uint2 *)(table + 2 * (uint64_t)(page0 + lane)) : make_uint2(0, 0);
  };
  uint2 entry = request_entry(first_page);
  // A row behind the causal limit of another has weight zero there, which a value of no number would turn into one.  Where the
  // batch brings such values, its own rows enter the sums with zeros for them, and the rows that attend them get them at the
  // end.  (What was cached before is attended by all.)
  const uint32_t new_from = p.starts[item.lane], clean_from = p.counts[4] == p.not_finite ? new_from : 0xffffffffu;
  // This lane's query row, and the keys of this wave's rows: none at or past wave_end, all below plain_end.
  const uint32_t rows = item.members * p.group, row = 32 * wave + (lane & 31);
  const bool used = row < rows;
  const uint32_t member = used ? row / p.group : 0, head = kv_head * p.group + (used ? row % p.group : 0);
  const uint32_t own_limit = !used ? 0 : min(end, item.attended + member);
  uint32_t wave_end = begin, plain_end = begin;
  if (32 * wave < rows) {
    const uint32_t last = (min(32 * wave + 32, rows) - 1) / p.group, first = 32 * wave / p.group;
    wave_end = min(end, item.attended + last);
    plain_end = min(end, item.attended + first);
  }
  const float scale_log2 = p.scale_log2 == 0.0f ? 1.0f : fabsf(p.scale_log2);
  RawQuery<kWide> raw[D / 32];   // (an unused row takes the unit's first: its keys are all masked and nothing of it is stored)
#pragma unroll
  for (int j = 0; j < D / 32; ++j)   // kWide: elements 32 j + 16 half on; else: 64 (j / 2) + 32 half + 16 (j % 2) on
    request_query<kWide>(p, (uint64_t)(item.leader + member) * p.q_stride_t + (uint64_t)head * p.q_stride_h +
                                (kWide ? 32 * j + 16 * half : 64 * (j / 2) + 32 * half + 16 * (j % 2)), raw[j]);
  PromptQueries<D, kWide> q;
  make_prompt_queries<D, kWide>(p, q, raw, p.scale_log2 == 0.0f ? 0.0f : copysignf(1.0f, p.scale_log2));
  f32x16 o[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = 0.0f;
  Softmax sm{-__builtin_inff(), 0.0f};
  const TilePlaces<D, kWide> places = tile_places<D, kWide>(tiles, p.kv_heads * D, wave, lane);
  for (uint32_t page0 = first_page; page0 <= last_page; page0 += 64) {
    // Nothing is dereferenced through an entry that is not authentic.
    const uint32_t my_page = page0 + lane, physical = entry.x;
    const bool mine = my_page <= last_page, ok = !mine || (physical < p.physical_pages && p.generations[physical] == entry.y);
    const unsigned long long bad_mask = __ballot(!ok);
    const uint32_t low = max(begin, page0 * pt);
    uint32_t high = (uint32_t)min((uint64_t)end, ((uint64_t)page0 + 64) * pt);
    if (bad_mask) {
      const uint32_t refused = page0 + (uint32_t)__ffsll((long long)bad_mask) - 1;
      refused_from = refused * pt;
      if (wave == 0 && my_page == refused) {
        report_error(error, refused);
        for (uint32_t m = refused_from >= item.attended ? refused_from - item.attended + 1 : 0; m < item.members; ++m) p.bad[item.leader + m] = 1;
      }
      if (refused_from <= low) break;
      last_page = refused - 1;
      high = refused_from;
      wave_end = min(wave_end, refused_from);
    }
    const uint32_t limit = min(own_limit, high), group_end = min(wave_end, high);
    const uint32_t start = min(low + 16 * wave, (high - 1) & ~15u);
    StageCursor at{start / pt - page0, start % pt};
    Arriving<D> in;
    request_tile<D, kWide>(p, in, places, 0, low, high, at, physical, kv_head, wave, lane);
    settle_tile<D, kWide>(in, places, 0, low, high, clean_from, wave, lane);
    // One tile out of `buffer`, while the next comes into `other` (constants, so that they are the instructions' offsets).
    auto step = [&](uint32_t tile0, uint32_t buffer, uint32_t other) {
      __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this wave's keys of the tile have landed
      __syncthreads();                      // everybody's share has, and the other buffer is free
      const uint32_t next0 = tile0 + kPromptTile;
      if (next0 < high) {
        if (next0 + 16 * wave < high) {
          at.slot += kPromptTile;
          while (at.slot >= pt) {
            at.slot -= pt;
            ++at.page;
          }
        }
        request_tile<D, kWide>(p, in, places, other, next0, high, at, physical, kv_head, wave, lane);
      }
      if (tile0 < group_end)
        attend_tile<D, kWide>(p, places, buffer, q, o, sm, next0 > min(plain_end, high), tile0, limit, scale_log2, lane);
      if (next0 < high) settle_tile<D, kWide>(in, places, other, next0, high, clean_from, wave, lane);
    };
    for (uint32_t tile0 = low; tile0 < high; tile0 += 2 * kPromptTile) {
      step(tile0, 0, S::kBytes);
      if (tile0 + kPromptTile < high) step(tile0 + kPromptTile, S::kBytes, 0);
    }
    entry = request_entry(page0 + 64);
    __syncthreads();   // the next tile staged goes into the first buffer
  }
  if (clean_from != 0xffffffffu) {
    wave_end = min(wave_end, refused_from);
    const uint32_t first_token = p.cu[item.lane], row_bytes = p.kv_heads * D;
    for (uint32_t base = max(begin, new_from); base < wave_end; base += 64) {
      const uint32_t mine = base + lane;
      const bool marked = mine < wave_end && p.not_finite_rows[first_token + (mine - new_from)] == p.not_finite;
      for (unsigned long long left = __ballot(marked); left != 0; left &= left - 1) {
        const uint32_t key = base + (uint32_t)__ffsll((long long)left) - 1;
        const uint8_t *codes = p.value_codes + ((uint64_t)table[2 * (uint64_t)(key / pt)] * pt + key % pt) * row_bytes + kv_head * D;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const uint32_t found = key < own_limit ? no_numbers(*(const uint32_t *)(codes + 32 * c + 8 * n + 4 * half)) : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (found >> (8 * i + 7) & 1) o[c][4 * n + i] = __builtin_nanf("");
          }
      }
    }
  }
  sm.l += __shfl_xor(sm.l, 32, 64);
  if (!used) return;
  // This lane holds value columns 32c + 8n + 4 * half + 0..3 of its row in o[c][4n..4n + 3].
  const bool single = item.splits == 1, zero = single && item.attended + member > refused_from;   // (of several splits the merge knows)
  const float inverse = single ? 1.0f / sm.l : 1.0f;
  const uint64_t slot = (uint64_t)(item.base + member * p.prompt_splits + item.split) * p.query_heads + head;
  const uint64_t to = (uint64_t)(item.leader + member) * p.out_stride_t + (uint64_t)head * p.out_stride_h;
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint32_t column = 32 * c + 8 * n + 4 * half;
      const float x = o[c][4 * n] * inverse, y = o[c][4 * n + 1] * inverse, z = o[c][4 * n + 2] * inverse, w = o[c][4 * n + 3] * inverse;
      if (single)
        store_out4(p, to + column, zero ? 0.0f : x, zero ? 0.0f : y, zero ? 0.0f : z, zero ? 0.0f : w);
      else
        *(float4 *)(p.partial_o + slot * D + column) = make_float4(x, y, z, w);
    }
  if (!single && half == 0) p.partial_ml[slot] = make_float2(sm.m, sm.l);
}

// A batch with prompt rows: the items of several tokens, the kv heads of an item side by side (with 8, 4, 2 or 1 kv heads
// a head's items then meet in the L2 of one XCD, as workgroups go to the XCDs in turn), and behind them those of one token,
// four waves of a kv head each.  What bounds it: instructions of both kinds, one wave's matrix products hardly running beside
// the other's softmax (matrix cores busy 49 %, vector ALUs 52 % of the time; raising a wave's priority over one or the other
// part changes nothing): 2048 rows behind 16384 keys, 32 heads, 629 us, 0.93 PFLOP/s; 8192 rows of 6 prompts and 64 lanes,
// 40 heads, 235 us, 0.57, where a unit's start (list, entries, first tile: 6 us) is as long as three tiles.  f32: 3 us a tile; heads of
// 128 then need more registers than there are (30 spilled, 116 bytes of scratch a lane, most of them around a unit's start and end).
template <int D, bool kWide>
__global__ __launch_bounds__(64 * kPromptWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void quant_prompt_kernel(QuantBatch p, ErrorSlot *error) {
  __shared__ uint4 tiles[2 * Staged<D>::kBytes / 16];
  const uint32_t prompts = p.counts[3], places = p.kv_heads * p.head_tiles, each = (places + kPromptWaves - 1) / kPromptWaves;
  const uint32_t listed = prompts * p.kv_heads, all = listed + (p.counts[0] - prompts) * each;
  for (uint32_t entry = blockIdx.x; entry < all; entry += gridDim.x) {
    if (entry < listed) {
      attend_unit<D, kWide>(p, error, lds_address(tiles), p.items[entry / p.kv_heads], entry % p.kv_heads);
    } else {
      const uint32_t place = (entry - listed) % each * kPromptWaves + (threadIdx.x >> 6);
      if (place < places) attend_token<D, kWide>(p, error, p.items[prompts + (entry - listed) / each], place / p.head_tiles, place % p.head_tiles);
    }
  }
}

// Merges the splits of a (token, head): out = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M); zero rows too.  Of many splits by a
// workgroup: a thread finds the weight of a split, then every D / 4 threads fold a stream of them, and the streams meet in
// LDS; where there are workgroups to spare, 64 columns to each (32 heads of one token of 235 splits 7.2 -> 6.2 us, 8 tokens of
// 32 splits 6.7 -> 5.9).  Of few (and zero rows) by D / 4 threads, one split after the other.  What bounds it: the chain list,
// weights, rows.  (4096 rows of two splits with 32 heads, a workgroup each: 109 us, as they are now 5; 32 rows of up to 32
// splits by D / 4 threads each: 15 us, now 5.)
template <int D, uint32_t kParts>
__device__ inline void merge_many(const QuantBatch &p, const uint4 &entry, uint32_t head, uint32_t part) {
  constexpr uint32_t kLanes = D / 4 / kParts, kStreams = kMergeThreads / kLanes, kWaves = kMergeThreads / 64, kHeld = 4;
  __shared__ float weights[kMostSplits], of_wave[2][kWaves];
  __shared__ float4 folded[kStreams][kLanes];
  const uint32_t thread = threadIdx.x, lane = thread & 63, wave = thread >> 6, column = (part * kLanes + thread % kLanes) * 4, stream = thread / kLanes;
  const uint32_t token = entry.x, splits = entry.y;
  const uint64_t base = (uint64_t)entry.z * p.query_heads + head;
  const bool refused = p.bad[token] != 0;
  float4 held[kHeld];   // the stream's first splits, requested before anything is known of their weights
#pragma unroll
  for (uint32_t i = 0; i < kHeld; ++i)
    if (stream + kStreams * i < splits)
      held[i] = *(const float4 *)(p.partial_o + (base + (uint64_t)(stream + kStreams * i) * p.query_heads) * D + column);
  // (waves without a split of theirs have nothing to add)
  const bool mine = 64 * wave < splits;
  float2 ml = make_float2(-__builtin_inff(), 0.0f);
  if (thread < splits) ml = p.partial_ml[base + (uint64_t)thread * p.query_heads];
  if (mine) {
    const float most = wave_max(ml.x);
    if (lane == 0) of_wave[0][wave] = most;
  }
  __syncthreads();   // (and the sums of the row before have been read)
  float m_all = of_wave[0][0];
  for (uint32_t w = 1; 64 * w < splits; ++w) m_all = fmaxf(m_all, of_wave[0][w]);
  if (mine) {
    const float weight = thread < splits && m_all > -__builtin_inff() ? exp2f(ml.x - m_all) : 0.0f;
    weights[thread] = weight;
    const float sum = wave_sum(ml.y * weight);
    if (lane == 0) of_wave[1][wave] = sum;
  }
  __syncthreads();
  float l_all = of_wave[1][0];
  for (uint32_t w = 1; 64 * w < splits; ++w) l_all += of_wave[1][w];
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto fold = [&](const float4 &one, float w) {
    acc.x += one.x * w;
    acc.y += one.y * w;
    acc.z += one.z * w;
    acc.w += one.w * w;
  };
#pragma unroll
  for (uint32_t i = 0; i < kHeld; ++i)
    if (stream + kStreams * i < splits) fold(held[i], weights[stream + kStreams * i]);
#pragma unroll 4
  for (uint32_t s = stream + kStreams * kHeld; s < splits; s += kStreams)
    fold(*(const float4 *)(p.partial_o + (base + (uint64_t)s * p.query_heads) * D + column), weights[s]);
  folded[stream][thread % kLanes] = acc;
  __syncthreads();
  if (thread < kLanes) {
    for (uint32_t other = 1; other < min(kStreams, splits); ++other) {
      const float4 one = folded[other][thread];
      acc.x += one.x;
      acc.y += one.y;
      acc.z += one.z;
      acc.w += one.w;
    }
    const float inverse = refused ? 0.0f : 1.0f / l_all;
    if (refused) acc = make_float4(0.f, 0.f, 0.f, 0.f);
    store_out4(p, (uint64_t)token * p.out_stride_t + (uint64_t)head * p.out_stride_h + column, acc.x * inverse, acc.y * inverse,
               acc.z * inverse, acc.w * inverse);
  }
}

template <int D>
__device__ inline void merge_few(const QuantBatch &p, const uint4 &entry, uint32_t head, uint32_t column) {
  const uint32_t token = entry.x, splits = entry.y;
  const uint64_t base = (uint64_t)entry.z * p.query_heads + head;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (splits != 0 && p.bad[token] == 0) {
    float2 ml[kFewSplits];
    float4 one[kFewSplits];
    float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
    for (uint32_t s = 0; s < kFewSplits; ++s) {
      if (s >= splits) continue;
      ml[s] = p.partial_ml[base + (uint64_t)s * p.query_heads];
      one[s] = *(const float4 *)(p.partial_o + (base + (uint64_t)s * p.query_heads) * D + column);
      m = fmaxf(m, ml[s].x);
    }
#pragma unroll
    for (uint32_t s = 0; s < kFewSplits; ++s) {
      if (s >= splits) continue;
      const float w = m > -__builtin_inff() ? exp2f(ml[s].x - m) : 0.0f;
      l += ml[s].y * w;
      acc.x += one[s].x * w;
      acc.y += one[s].y * w;
      acc.z += one[s].z * w;
      acc.w += one[s].w * w;
    }
    const float inverse = 1.0f / l;
    acc = make_float4(acc.x * inverse, acc.y * inverse, acc.z * inverse, acc.w * inverse);
  }
  store_out4(p, (uint64_t)token * p.out_stride_t + (uint64_t)head * p.out_stride_h + column, acc.x, acc.y, acc.z, acc.w);
}

template <int D>
__global__ __launch_bounds__(kMergeThreads) void quant_merge_kernel(QuantBatch p) {
  constexpr uint32_t kLanes = D / 4, kRows = kMergeThreads / kLanes;
  const uint32_t many = p.counts[1] * p.query_heads;
  constexpr uint32_t kParts = D / 64;   // (of 32 columns: no faster)
  const uint32_t shared = kParts * many <= gridDim.x ? kParts * many : many;
  if (shared != many) {
    if (blockIdx.x < shared) merge_many<D, kParts>(p, p.merge[blockIdx.x / kParts / p.query_heads], blockIdx.x / kParts % p.query_heads, blockIdx.x % kParts);
  } else {
    for (uint32_t row = blockIdx.x; row < many; row += gridDim.x)
      merge_many<D, 1>(p, p.merge[row / p.query_heads], row % p.query_heads, 0);
  }
  // the workgroups that had none of those come first
  const uint32_t few = p.counts[5] * p.query_heads, place = (blockIdx.x + gridDim.x - shared % gridDim.x) % gridDim.x;
  for (uint32_t row = place * kRows + threadIdx.x / kLanes; row < few; row += gridDim.x * kRows)
    merge_few<D>(p, p.merge[p.tokens - 1 - row / p.query_heads], row % p.query_heads, threadIdx.x % kLanes * 4);
}

// ---- host side of the fast form ----

uint64_t round_256(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

using BatchKernel = void (*)(QuantBatch, ErrorSlot *);

BatchKernel decode_kernel(uint32_t width, bool wide) {
  if (width == 64) return wide ? quant_decode_kernel<64, true> : quant_decode_kernel<64, false>;
  return wide ? quant_decode_kernel<128, true> : quant_decode_kernel<128, false>;
}

BatchKernel prompt_kernel(uint32_t width, bool wide) {
  if (width == 64) return wide ? quant_prompt_kernel<64, true> : quant_prompt_kernel<64, false>;
  return wide ? quant_prompt_kernel<128, true> : quant_prompt_kernel<128, false>;
}

// Workgroups of `kernel` that a compute unit holds; asked once a kernel, by whichever backend's thread comes first (others
// that ask meanwhile store the same value).
uint32_t resident(BatchKernel kernel, uint32_t threads, std::atomic<uint32_t> *known) {
  uint32_t held = known->load(std::memory_order_relaxed);
  if (held == 0) {
    int blocks = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, (int)threads, 0) != hipSuccess || blocks < 1) {
      (void)hipGetLastError();
      blocks = 1;
    }
    held = (uint32_t)blocks;
    known->store(held, std::memory_order_relaxed);
  }
  return held;
}

bool fast_eligible(const RaggedQuantAttention &p) {
  if (p.width != p.value_width || (p.width != 64 && p.width != 128) || p.page_tokens % 16) return false;
  if (p.lanes > kPlanLanes || (uint64_t)p.kv_heads * p.width > (1u << 26)) return false;
  if (p.q.stride[2] != 1 || p.q.stride[0] % 8 || p.q.stride[1] % 8 || p.q.offset % 8) return false;
  if (p.out.stride[2] != 1 || p.out.stride[0] % 4 || p.out.stride[1] % 4 || p.out.offset % 4) return false;
  if (p.query_heads / p.kv_heads > kPromptRows || p.physical_pages == 0) return false;
  return p.key_codes.offset % 4 == 0 && p.value_codes.offset % 4 == 0;
}

// False when workspace allocation fails.
bool run_fast(fh_backend *backend, const RaggedQuantAttention &p, ErrorSlot *error) {
  hipStream_t stream = backend_stream(backend);
  QuantBatch f{};
  auto at = [](const View &v) { return (char *)v.base + v.offset * dtype_size(v.dtype); };
  f.q = at(p.q);
  f.k_new = at(p.k_new);
  f.v_new = at(p.v_new);
  f.out = at(p.out);
  f.key_codes = (uint8_t *)at(p.key_codes);
  f.value_codes = (uint8_t *)at(p.value_codes);
  f.scales = (uint8_t *)at(p.scales);
  f.tables = (const uint32_t *)at(p.tables);
  f.generations = (const uint32_t *)at(p.generations);
  f.cu = (const uint32_t *)at(p.cu_seqlens);
  f.starts = (const uint32_t *)at(p.q_starts);
  f.activity = p.activity.base ? (const uint32_t *)at(p.activity) : nullptr;
  f.q_stride_t = p.q.stride[0];
  f.q_stride_h = p.q.stride[1];
  f.out_stride_t = p.out.stride[0];
  f.out_stride_h = p.out.stride[1];
  f.kn_stride_t = p.k_new.stride[0];
  f.kn_stride_h = p.k_new.stride[1];
  f.vn_stride_t = p.v_new.stride[0];
  f.vn_stride_h = p.v_new.stride[1];
  f.q_dtype = p.q.dtype;
  f.out_dtype = p.out.dtype;
  f.tokens = p.tokens;
  f.lanes = p.lanes;
  f.query_heads = p.query_heads;
  f.kv_heads = p.kv_heads;
  f.group = p.query_heads / p.kv_heads;
  f.head_tiles = (f.group + 15) / 16;
  f.page_tokens = p.page_tokens;
  f.scale_bytes = 4 * p.scale_words;
  f.physical_pages = p.physical_pages;
  f.table_pages = p.table_pages;
  f.scale_log2 = p.scale * 1.4426950408889634f;
  f.promised = p.one_row_per_lane;
  // (a launch of its own takes 4 us a layer, and the attention is no faster for it)
  f.append_in_kernel = p.one_row_per_lane && f.head_tiles == 1 && p.k_new.stride[2] == 1 && p.v_new.stride[2] == 1;
  const bool wide = p.q.dtype != FH_BF16 || p.out.dtype == FH_F32;
  // Rows beyond the lanes: some lane brings several.  (Under the promise of one row a lane, they belong to none.)  Attended a
  // token at a time 8 lanes of 12 rows behind 4000 keys take 74 us instead of 27, 2048 rows and 32 lanes 474 instead of 92.
  const bool prompts = p.tokens > p.lanes && !p.one_row_per_lane;
  f.prompt_tokens = prompts ? kPromptRows / f.group : 0;
  const uint32_t places = f.kv_heads * f.head_tiles, waves = prompts ? kPromptWaves : std::min(places, 8u);
  const uint32_t per_item = (places + waves - 1) / waves;
  BatchKernel kernel = prompts ? prompt_kernel(p.width, wide) : decode_kernel(p.width, wide);
  static std::atomic<uint32_t> known[2][2][2][9];   // [width][wide][prompts][waves]
  const uint32_t held = resident(kernel, 64 * waves, &known[p.width / 128][wide][prompts][waves]);
  f.item_slots = std::max(held * backend_compute_units(backend) / per_item, 1u);
  // Partial slots: of the tokens, or of the lanes that bring one and of the tokens of others; none of a unit that is not split.
  const uint32_t singles = prompts ? f.lanes : f.tokens;
  f.max_splits = std::max(1u, std::min(kMostSplits, (prompts ? 8192u : 16384u) / singles));
  f.prompt_splits = prompts ? std::max(1u, std::min(64u, 8192u / f.tokens)) : 0;
  const uint64_t row_bytes = (uint64_t)f.query_heads * p.width * sizeof(float);
  auto slots = [&] {
    f.single_slots = f.max_splits > 1 ? singles * f.max_splits : 0;
    return f.single_slots + (f.prompt_splits > 1 ? (uint64_t)f.tokens * f.prompt_splits : 0);
  };
  auto ml_bytes = [&] { return round_256(slots() * f.query_heads * sizeof(float2)); };
  auto partial_bytes = [&] { return ml_bytes() + slots() * row_bytes + 256; };   // (never nothing: a null workspace is a refused one)
  while (partial_bytes() > backend_workspace_limit(backend) && (f.max_splits > 1 || f.prompt_splits > 1)) {
    if (f.max_splits >= f.prompt_splits)
      --f.max_splits;
    else
      --f.prompt_splits;
  }
  // The plan depends on the lane metadata only, which every layer of a step shares: it is built by the first attention
  // dispatch of a submission and reused until that metadata is written.
  AttentionPlanKey key{};
  for (int i = 0; i < 5; ++i) key.buffers[i] = p.metadata_buffers[i];
  const void *const addresses[5] = {f.cu, f.starts, f.activity, f.tables, f.generations};
  for (int i = 0; i < 5; ++i) key.address[i] = (uint64_t)addresses[i];
  const uint32_t params[14] = {f.tokens, f.lanes, f.page_tokens, f.physical_pages, f.table_pages, f.max_splits, f.promised,
                               f.item_slots, f.prompt_tokens, f.prompt_splits, f.kv_heads, 0, 0, 2 /* not a plan of the 16-bit kernels, which have 0 or 1 here */};
  for (int i = 0; i < 14; ++i) key.params[i] = params[i];
  const uint64_t words = round_256((uint64_t)f.tokens * 4);
  // (units of several tokens: one a lane at most is not whole)
  const uint64_t prompt_units = prompts ? f.tokens / f.prompt_tokens + f.lanes : 0;
  const uint64_t items = (uint64_t)singles * f.max_splits + prompt_units * f.prompt_splits;
  const uint64_t item_bytes = round_256(items * sizeof(QuantItem));
  bool reuse = false;
  char *plan = backend_attention_plan(backend, key, 8 * words + item_bytes + 256, &reuse);
  char *workspace = plan ? backend_workspace(backend, partial_bytes()) : nullptr;
  if (!workspace) return false;
  f.bad = (uint32_t *)plan;
  f.not_finite_rows = (uint32_t *)(plan + words);
  f.tokens_of = (uint2 *)(plan + 2 * words);
  f.merge = (uint4 *)(plan + 4 * words);
  f.items = (QuantItem *)(plan + 8 * words);
  f.counts = (uint32_t *)(plan + 8 * words + item_bytes);
  f.partial_ml = (float2 *)workspace;
  f.partial_o = (float *)(workspace + ml_bytes());
  const uint64_t rows = (uint64_t)p.tokens * 2 * p.kv_heads;
  const bool pieces = in_pieces(p.k_new, p.width) && in_pieces(p.v_new, p.width);
  // a word of its own for every launch says that it met a row that is not finite: nothing has to be cleared
  static std::atomic<uint32_t> launches{0};
  f.not_finite = ++launches;
  if (!reuse) {
    // The plan, and beside it the new rows: the attention then finds them stored.
    if (pieces) f.append_in_kernel = false;
    auto prepare = [&](auto *of_64, auto *of_128, uint32_t each) {
      const uint32_t tokens = each / 64, most = backend_compute_units(backend) * 2048 / each;   // what the device holds at once
      const dim3 grid(1 + (pieces ? std::min((f.tokens + tokens - 1) / tokens, most) : 0));
      (p.width == 64 ? of_64 : of_128)<<<grid, each, 0, stream>>>(f, error);
    };
    // A barrier of a larger workgroup costs more (48 lanes: 256 threads 6.4 us, 1024 threads 8.3; one wave is no faster: one lane
    // 5.2 us); many units need its threads (8256 tokens of 70 lanes: 15 us of plan beside 15 of storing, in 25).
    if (f.lanes <= 256 && f.tokens <= 1024)
      prepare(quant_prepare_kernel<256, 8>, quant_prepare_kernel<256, 16>, 256);
    else
      prepare(quant_prepare_kernel<1024, 8>, quant_prepare_kernel<1024, 16>, 1024);
  } else if (!f.append_in_kernel && pieces) {
    const dim3 grid((f.tokens + 1) / 2);
    (p.width == 64 ? quant_append_rows_kernel<8> : quant_append_rows_kernel<16>)<<<grid, 256, 0, stream>>>(f, error);
  }
  if (!f.append_in_kernel && !pieces)
    quant_append_kernel<<<dim3((unsigned)((rows + 3) / 4)), 256, 0, stream>>>(p, error, f.counts + 2, f.counts + 4, f.not_finite_rows,
                                                                              f.not_finite);
  {
    KernelTimer timer(backend, FH_KC_ATTENTION_KERNEL);
    if (prompts) {
      // what is left of the items' list, whose length only the device knows, the workgroups walk on
      const uint64_t entries = prompt_units * f.prompt_splits * f.kv_heads + (uint64_t)singles * f.max_splits * per_item;
      const uint64_t most = (uint64_t)kPromptGrid * backend_compute_units(backend);
      kernel<<<dim3((unsigned)std::min(entries, most)), 64 * waves, 0, stream>>>(f, error);
    } else {
      kernel<<<dim3((unsigned)std::min<uint64_t>(items, 2 * (uint64_t)f.item_slots), per_item), 64 * waves, 0, stream>>>(f, error);
    }
  }
  // Only the device knows how many rows there are to merge: at most as many workgroups as it holds, an empty one costs its place.
  const dim3 merge((unsigned)std::min<uint64_t>((uint64_t)f.tokens * f.query_heads * (p.width / 64), 8 * backend_compute_units(backend)));
  if (p.width == 64)
    quant_merge_kernel<64><<<merge, kMergeThreads, 0, stream>>>(f);
  else
    quant_merge_kernel<128><<<merge, kMergeThreads, 0, stream>>>(f);
  return true;
}

}  // namespace

void run_quant_copy(fh_backend *backend, const QuantCopy &p, bool into_pages, ErrorSlot *error) {
  const uint64_t rows = (uint64_t)p.tokens * p.heads;
  if (rows == 0) return;
  hipStream_t stream = backend_stream(backend);
  const bool pieces = in_pieces(p.rows, 4 * p.words) && p.codes.offset % 2 == 0;
  const dim3 whole((unsigned)((rows * (p.words / 2) + 255) / 256));
  if (into_pages && pieces && p.words == 16)
    quant_store_rows_kernel<8><<<whole, 256, 0, stream>>>(p, error);
  else if (into_pages && pieces && p.words == 32)
    quant_store_rows_kernel<16><<<whole, 256, 0, stream>>>(p, error);
  else if (into_pages && pieces && p.words == 64)
    quant_store_rows_kernel<32><<<whole, 256, 0, stream>>>(p, error);
  else if (into_pages)
    quant_store_kernel<<<dim3((unsigned)((rows + 3) / 4)), 256, 0, stream>>>(p, error);
  else if (pieces)
    quant_load_rows_kernel<<<whole, 256, 0, stream>>>(p, error);
  else
    quant_load_kernel<<<dim3((unsigned)((rows * p.words + 255) / 256)), 256, 0, stream>>>(p, error);
}

bool run_quant_attention(fh_backend *backend, const RaggedQuantAttention &p, ErrorSlot *error) {
  if (fast_eligible(p)) return run_fast(backend, p, error);
  hipStream_t stream = backend_stream(backend);
  uint32_t *malformed = (uint32_t *)backend_workspace(backend, 256);
  if (!malformed) return false;
  quant_validate_kernel<<<dim3(1), 256, 0, stream>>>((const uint32_t *)p.cu_seqlens.base + p.cu_seqlens.offset, p.lanes,
                                                     p.tokens, malformed, error);
  const uint64_t rows = (uint64_t)p.tokens * 2 * p.kv_heads;
  quant_append_kernel<<<dim3((unsigned)((rows + 3) / 4)), 256, 0, stream>>>(p, error, malformed, nullptr, nullptr, 0);
  const dim3 grid(p.tokens * p.query_heads);
  if (p.value_width <= 64)
    quant_attention_generic_kernel<16><<<grid, 64, 0, stream>>>(p, error, malformed);
  else if (p.value_width <= 128)
    quant_attention_generic_kernel<32><<<grid, 64, 0, stream>>>(p, error, malformed);
  else
    quant_attention_generic_kernel<64><<<grid, 64, 0, stream>>>(p, error, malformed);
  return true;
}

}  // namespace fh
