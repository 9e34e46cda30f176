// One step of batched serving through the C++ mirror (include/kraken/hip_context.hpp):
// two sequences append their first token to pages, attend it, the pages are read back and
// a token is drawn for each.
//
//   paged_check cpu   no GPU needed: a validation-only context refuses and accepts
//   paged_check gpu   closed forms: a token that sees itself alone gets its own value, as
//                     the page holds it, times the gate's sigmoid; top-k 1 draws the
//                     largest logit
// Prints one line per check and exits non-zero if one failed.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "kraken/hip_context.hpp"

using kraken::hip::HipBuffer;
using kraken::hip::HipContext;
using kraken::hip::Status;
using kraken::hip::StatusCode;

namespace {

constexpr std::size_t kPages = 3, kPageTokens = 16, kKvHeads = 2, kHeads = 4, kDim = 64;
constexpr std::size_t kSequences = 2, kVocabulary = 1000;

int failures = 0;

void expect(bool ok, const std::string& what, const Status& s = Status::ok()) {
  std::printf("%s %s%s%s\n", ok ? "ok  " : "FAIL", what.c_str(), s.message().empty() ? "" : ": ",
              s.message().c_str());
  if (!ok) {
    ++failures;
  }
}

struct Buffers {
  HipBuffer keys, values, key_scales, value_scales, table, starts, lengths;

  kraken_paged_q8_cache cache() const {
    return {keys.raw(), values.raw(), key_scales.raw(), value_scales.raw(), kPages,
            kPageTokens, kKvHeads, kDim};
  }
  kraken_paged_batch batch() const {
    return {table.raw(), starts.raw(), lengths.raw(), kSequences, 1, kSequences, 1, kPageTokens};
  }
};

HipBuffer fake(std::size_t bytes) {
  return HipBuffer::borrow(reinterpret_cast<void*>(std::uintptr_t{4096}), bytes);
}

int run_cpu() {
  auto made = HipContext::create_validation_only();
  expect(made.is_ok(), "a validation context is made", made.status());
  if (!made.is_ok()) {
    return 1;
  }
  const HipContext& ctx = made.value();
  const std::size_t codes = kPages * kKvHeads * kPageTokens * kDim, scales = kPages * kKvHeads * 4;
  Buffers b{fake(codes), fake(codes), fake(scales), fake(scales), fake(8), fake(12), fake(8)};
  HipBuffer out = fake(kSequences * kHeads * kDim * 4);
  const HipBuffer query = fake(kSequences * kHeads * kDim * 4);
  Status s = ctx.attention_f32_paged_q8_kv(query, HipBuffer(), b.cache(), b.batch(), kHeads, out);
  expect(s.code() == StatusCode::unavailable, "attention accepts its arguments", s);
  s = ctx.attention_f16q_paged_q8_kv(query, b.cache(), b.batch(), 3, out);
  expect(s.code() == StatusCode::invalid_argument, "heads % kv_heads != 0 refused", s);
  b.keys = fake(codes - 1);
  s = ctx.dequantize_kv_pages_q8_f16(b.cache(), fake(4), 1, out, out);
  expect(s.code() == StatusCode::invalid_argument, "a short page pool refused", s);
  HipBuffer token = fake(8), none;
  s = ctx.sample_f32_i32(fake(8 * kVocabulary), 2, kVocabulary, kVocabulary, none, none, none,
                         none, fake(8), token, none);
  expect(s.code() == StatusCode::unavailable, "sampling accepts its arguments", s);
  s = ctx.sample_f32_i32(fake(8 * kVocabulary), 2, kVocabulary, kVocabulary - 1, none, none, none,
                         none, fake(8), token, none);
  expect(s.code() == StatusCode::invalid_argument, "a row stride below the size refused", s);
  return failures;
}

float from_half(std::uint16_t h) {
  const float mantissa = (float)(h & 0x3ffu) / 1024.0f;
  const int exponent = (h >> 10) & 0x1f;
  const float x = exponent == 0 ? std::ldexp(mantissa, -14)
                                : std::ldexp(1.0f + mantissa, exponent - 15);
  return (h & 0x8000u) != 0 ? -x : x;
}

template <class T>
HipBuffer upload(const HipContext& ctx, const std::vector<T>& x) {
  auto made = ctx.make_buffer(x.size() * sizeof(T));
  expect(made.is_ok(), "a buffer of " + std::to_string(x.size()), made.status());
  HipBuffer b = std::move(made.value());
  const Status s = ctx.copy_to_buffer(b, x.data(), x.size() * sizeof(T));
  if (!s.is_ok()) {
    expect(false, "its copy", s);
  }
  return b;
}

template <class T>
std::vector<T> download(const HipContext& ctx, const HipBuffer& b) {
  std::vector<T> x(b.byte_size() / sizeof(T));
  const Status s = ctx.copy_from_buffer(b, x.data(), x.size() * sizeof(T));
  if (!s.is_ok()) {
    expect(false, "a copy back", s);
  }
  return x;
}

int run_gpu() {
  auto made = HipContext::create();
  expect(made.is_ok(), "a context is made", made.status());
  if (!made.is_ok()) {
    return 1;
  }
  const HipContext& ctx = made.value();
  const std::size_t codes = kPages * kKvHeads * kPageTokens * kDim;
  Buffers b{upload(ctx, std::vector<std::int8_t>(codes, 5)),
            upload(ctx, std::vector<std::int8_t>(codes, 5)),
            upload(ctx, std::vector<float>(kPages * kKvHeads, NAN)),
            upload(ctx, std::vector<float>(kPages * kKvHeads, NAN)),
            upload(ctx, std::vector<std::int32_t>{2, 0}),
            upload(ctx, std::vector<std::uint32_t>{0, 1, 2}),
            upload(ctx, std::vector<std::uint32_t>{1, 1})};
  std::vector<float> q_gate(kSequences * kHeads * 2 * kDim), kv(kSequences * kKvHeads * kDim);
  for (std::size_t i = 0; i < q_gate.size(); ++i) {
    q_gate[i] = std::sin(0.37f * (float)i);
  }
  for (std::size_t i = 0; i < kv.size(); ++i) {
    kv[i] = std::cos(0.11f * (float)i);
  }
  const HipBuffer w = upload(ctx, std::vector<float>(kDim, 1.0f));
  const std::size_t rows = kSequences * kHeads * kDim;
  HipBuffer query = upload(ctx, std::vector<float>(rows));
  HipBuffer gate = upload(ctx, std::vector<float>(rows));
  HipBuffer out = upload(ctx, std::vector<float>(rows));
  Status s = ctx.qwen35_attention_prologue_paged_q8_kv(
    upload(ctx, q_gate), upload(ctx, kv), upload(ctx, kv), w, w, HipBuffer(), b.cache(), b.batch(),
    kHeads, kDim, 8, 8, 8, 8, 1e6f, 1e-6f, query, gate);
  expect(s.is_ok(), "the prologue appends", s);
  s = ctx.attention_f32_paged_q8_kv(query, gate, b.cache(), b.batch(), kHeads, out);
  expect(s.is_ok(), "attention runs", s);
  const std::size_t page = kPageTokens * kKvHeads * kDim;
  HipBuffer key_rows = upload(ctx, std::vector<std::uint16_t>(2 * page));
  HipBuffer value_rows = upload(ctx, std::vector<std::uint16_t>(2 * page));
  s = ctx.dequantize_kv_pages_q8_f16(b.cache(), upload(ctx, std::vector<std::int32_t>{2, 0}), 2,
                                     key_rows, value_rows);
  expect(s.is_ok(), "the pages are read back", s);
  const auto got = download<float>(ctx, out), g = download<float>(ctx, gate);
  const auto held = download<std::uint16_t>(ctx, value_rows);
  double off = 0, step = 0;
  for (std::size_t t = 0; t < kSequences; ++t) {
    for (std::size_t h = 0; h < kHeads; ++h) {
      for (std::size_t d = 0; d < kDim; ++d) {
        const std::size_t at = (t * kHeads + h) * kDim + d, kv_head = h / (kHeads / kKvHeads);
        const double value = kv[(t * kKvHeads + kv_head) * kDim + d];
        const double page_value = from_half(held[t * page + kv_head * kDim + d]);
        // Half a step of the largest value's 127th, and of f16.
        step = std::fmax(step, std::fabs(page_value - value));
        const double want = page_value / (1.0 + std::exp(-(double)g[at]));
        // Half a step of f16 (of values up to 1), and a few of f32.
        off = std::fmax(off, std::fabs(got[at] - want));
      }
    }
  }
  expect(step <= 0.5 / 127 * 1.001 + 0x1p-12, "a page holds its values to half a step");
  expect(off <= 0x1p-12 + 0x1p-20, "a token alone gets its own value times the gate");

  std::vector<float> logits(2 * kVocabulary);
  for (std::size_t i = 0; i < logits.size(); ++i) {
    logits[i] = std::sin(0.7f * (float)i);
  }
  logits[321] = 3.0f;
  logits[kVocabulary + 999] = 3.0f;
  HipBuffer token = upload(ctx, std::vector<std::int32_t>{-1, -1}), none;
  s = ctx.sample_f32_i32(upload(ctx, logits), 2, kVocabulary, kVocabulary, none,
                         upload(ctx, std::vector<std::int32_t>{1, 1}), none, none,
                         upload(ctx, std::vector<float>{0.9f, 0.0f}), token, none);
  expect(s.is_ok(), "sampling runs", s);
  const auto drawn = download<std::int32_t>(ctx, token);
  expect(drawn[0] == 321 && drawn[1] == 999, "top-k 1 draws the largest logit");
  return failures;
}

}  // namespace

int main(int argc, char** argv) {
  const std::string mode = argc > 1 ? argv[1] : "cpu";
  const int failed = mode == "gpu" ? run_gpu() : run_cpu();
  std::printf(failed == 0 ? "all checks passed\n" : "%d checks failed\n", failed);
  return failed == 0 ? 0 : 1;
}
