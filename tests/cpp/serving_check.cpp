// Shared prefixes, eviction by received attention and log probabilities through the C++
// mirror (include/kraken/hip_context.hpp).
//
//   serving_check cpu   no GPU needed: a validation-only context refuses and accepts
//   serving_check gpu   closed forms: zero queries weigh their keys alike, so that each key
//                       receives one share a row and a row's output is its values' mean;
//                       the cache then keeps its ends, and its pages their codes; of equal
//                       logits every token's share is the same
// Prints one line per check and exits non-zero if one failed.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <string>
#include <vector>

#include "kraken/hip_context.hpp"

using kraken::hip::HipBuffer;
using kraken::hip::HipContext;
using kraken::hip::Status;
using kraken::hip::StatusCode;

namespace {

constexpr std::size_t kPages = 8, kPageTokens = 16, kKvHeads = 2, kHeads = 4, kDim = 64;
constexpr std::size_t kSequences = 2, kWidth = 3, kLength = 40, kKeep = 12;

int failures = 0;

void expect(bool ok, const std::string& what, const Status& s = Status::ok()) {
  std::printf("%s %s%s%s\n", ok ? "ok  " : "FAIL", what.c_str(), s.message().empty() ? "" : ": ",
              s.message().c_str());
  if (!ok) {
    ++failures;
  }
}

struct Buffers {
  HipBuffer keys, values, key_scales, value_scales, table, starts, lengths, group_starts, prefixes;

  kraken_paged_q8_cache cache() const {
    return {keys.raw(), values.raw(), key_scales.raw(), value_scales.raw(), kPages,
            kPageTokens, kKvHeads, kDim};
  }
  kraken_paged_batch batch() const {
    return {table.raw(), starts.raw(), lengths.raw(), kSequences, kWidth, kSequences, 1, kLength};
  }
  kraken_shared_prefixes shared() const {
    return {group_starts.raw(), prefixes.raw(), 1, kSequences, 2 * kPageTokens};
  }
};

// Addresses that nothing reads, each buffer its own.
HipBuffer fake(std::size_t bytes) {
  static std::uintptr_t next = 4096;
  const std::uintptr_t at = next;
  next += (bytes + 4095) / 4096 * 4096;
  return HipBuffer::borrow(reinterpret_cast<void*>(at), bytes);
}

int run_cpu() {
  auto made = HipContext::create_validation_only();
  expect(made.is_ok(), "a validation context is made", made.status());
  if (!made.is_ok()) {
    return 1;
  }
  const HipContext& ctx = made.value();
  const std::size_t codes = kPages * kKvHeads * kPageTokens * kDim, scales = kPages * kKvHeads * 4;
  Buffers b{fake(codes), fake(codes), fake(scales), fake(scales), fake(24),
            fake(12), fake(8), fake(8), fake(4)};
  const std::size_t rows = kSequences * kHeads * kDim * 4;
  HipBuffer out = fake(rows), none;
  Status s = ctx.attention_f32_shared_paged_q8_kv(fake(rows), none, b.cache(), b.batch(),
                                                  b.shared(), kHeads, out);
  expect(s.code() == StatusCode::unavailable, "shared attention accepts its arguments", s);
  b.prefixes = fake(3);
  s = ctx.attention_f16q_shared_paged_q8_kv(fake(rows), b.cache(), b.batch(), b.shared(), kHeads,
                                            out);
  expect(s.code() == StatusCode::invalid_argument, "short prefix lengths refused", s);
  HipBuffer weights = fake(kSequences * kKvHeads * kLength * 4);
  s = ctx.key_weights_f32_paged_q8_kv(fake(rows), b.cache(), b.batch(), kHeads, 0, 1.0f, weights,
                                      kLength);
  expect(s.code() == StatusCode::unavailable, "key weights accept their arguments", s);
  s = ctx.key_weights_f16q_paged_q8_kv(fake(rows), b.cache(), b.batch(), kHeads, 0, -1.0f, weights,
                                       kLength);
  expect(s.code() == StatusCode::invalid_argument, "a negative decay refused", s);
  HipBuffer kept = fake(kSequences * kKvHeads * kKeep * 4), kept_lengths = fake(8);
  s = ctx.select_keys_f32_i32(weights, kLength, fake(8), fake(8), kSequences, kKvHeads, kLength,
                              1, 1, kept, kKeep, kept_lengths);
  expect(s.code() == StatusCode::unavailable, "the selection accepts its arguments", s);
  s = ctx.gather_kv_pages_q8(b.cache(), fake(24), kWidth, kept, kept_lengths, kKeep, kSequences,
                             fake(8), 1, weights, kLength, weights);
  expect(s.code() == StatusCode::invalid_argument, "weights gathered in place refused", s);
  HipBuffer value = fake(8);
  s = ctx.token_logprobs_f32(fake(800), 2, 100, 100, none, fake(8), 0, value, none, none, none,
                             none);
  expect(s.code() == StatusCode::unavailable, "log probabilities accept their arguments", s);
  s = ctx.token_logprobs_f32(fake(800), 2, 100, 100, none, fake(8), 33, value, none, none, value,
                             none);
  expect(s.code() == StatusCode::invalid_argument, "a list of 33 tokens refused", s);
  return failures;
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

std::int8_t key_code(std::size_t page, std::size_t head, std::size_t slot, std::size_t dim) {
  return static_cast<std::int8_t>((page * 37 + head * 11 + slot * 5 + dim) % 255);
}

int run_gpu() {
  auto made = HipContext::create();
  expect(made.is_ok(), "a context is made", made.status());
  if (!made.is_ok()) {
    return 1;
  }
  const HipContext& ctx = made.value();
  const std::size_t codes = kPages * kKvHeads * kPageTokens * kDim;
  std::vector<std::int8_t> keys(codes);
  for (std::size_t i = 0; i < codes; ++i) {
    const int code = key_code(i / (kKvHeads * kPageTokens * kDim),
                              i / (kPageTokens * kDim) % kKvHeads, i / kDim % kPageTokens, i % kDim);
    keys[i] = static_cast<std::int8_t>(code == -128 ? 0 : code);
  }
  // Two sequences of 40 tokens over the same first two pages.
  Buffers b{upload(ctx, keys),
            upload(ctx, std::vector<std::int8_t>(codes, 8)),
            upload(ctx, std::vector<float>(kPages * kKvHeads, 0.25f)),
            upload(ctx, std::vector<float>(kPages * kKvHeads, 0.25f)),
            upload(ctx, std::vector<std::int32_t>{4, 1, 2, 4, 1, 6}),
            upload(ctx, std::vector<std::uint32_t>{0, 1, 2}),
            upload(ctx, std::vector<std::uint32_t>{kLength, kLength}),
            upload(ctx, std::vector<std::uint32_t>{0, kSequences}),
            upload(ctx, std::vector<std::uint32_t>{2 * kPageTokens})};
  const HipBuffer query = upload(ctx, std::vector<float>(kSequences * kHeads * kDim));
  HipBuffer out = upload(ctx, std::vector<float>(kSequences * kHeads * kDim)), none;
  Status s = ctx.attention_f32_shared_paged_q8_kv(query, none, b.cache(), b.batch(), b.shared(),
                                                  kHeads, out);
  expect(s.is_ok(), "shared attention runs", s);
  double off = 0;
  for (const float x : download<float>(ctx, out)) {
    off = std::fmax(off, std::fabs(x - 2.0));
  }
  expect(off <= 2 * 0x1p-18, "a zero query takes the mean of equal values");

  HipBuffer weights = upload(ctx, std::vector<float>(kSequences * kKvHeads * kLength, 1.0f));
  s = ctx.key_weights_f32_paged_q8_kv(query, b.cache(), b.batch(), kHeads, 0, 0.5f, weights,
                                      kLength);
  expect(s.is_ok(), "key weights run", s);
  const auto received = download<float>(ctx, weights);
  off = 0;
  for (std::size_t i = 0; i < received.size(); ++i) {
    // Two heads' shares of one in forty, beside half of the one before.
    const double want = 2.0 / kLength + (i % kLength + 1 < kLength ? 0.5 : 0.0);
    off = std::fmax(off, std::fabs(received[i] - want));
  }
  expect(off <= 0x1p-20, "each key receives one share of each row");

  HipBuffer kept = upload(ctx, std::vector<std::int32_t>(kSequences * kKvHeads * kKeep, -1));
  HipBuffer kept_lengths = upload(ctx, std::vector<std::uint32_t>(kSequences));
  s = ctx.select_keys_f32_i32(upload(ctx, std::vector<float>(received.size(), 1.0f)), kLength,
                              b.lengths, upload(ctx, std::vector<std::uint32_t>{kKeep, kKeep}),
                              kSequences, kKvHeads, kLength, 2, 3, kept, kKeep, kept_lengths);
  expect(s.is_ok(), "the selection runs", s);
  const auto positions = download<std::int32_t>(ctx, kept);
  bool right = true;
  for (std::size_t i = 0; i < positions.size(); ++i) {
    const std::size_t at = i % kKeep;
    right = right && positions[i] == (std::int32_t)(at < kKeep - 3 ? at : kLength - kKeep + at);
  }
  expect(right, "equal weights keep the ends and the lowest positions");
  HipBuffer moved = upload(ctx, std::vector<float>(received.size(), -1.0f));
  s = ctx.gather_kv_pages_q8(b.cache(), b.table, kWidth, kept, kept_lengths, kKeep, kSequences,
                             upload(ctx, std::vector<std::int32_t>{0, 3}), 1, weights, kLength,
                             moved);
  expect(s.is_ok(), "the gather runs", s);
  const auto after = download<std::int8_t>(ctx, b.keys);
  const std::size_t sources[2][3] = {{4, 1, 2}, {4, 1, 6}}, targets[2] = {0, 3};
  right = true;
  for (std::size_t q = 0; q < kSequences; ++q) {
    for (std::size_t h = 0; h < kKvHeads; ++h) {
      for (std::size_t i = 0; i < kKeep; ++i) {
        const std::size_t j = (std::size_t)positions[(q * kKvHeads + h) * kKeep + i];
        for (std::size_t d = 0; d < kDim; ++d) {
          const auto at = [&](std::size_t page, std::size_t slot) {
            return ((page * kKvHeads + h) * kPageTokens + slot) * kDim + d;
          };
          right = right && after[at(targets[q], i)] ==
                             keys[at(sources[q][j / kPageTokens], j % kPageTokens)];
        }
      }
    }
  }
  expect(right, "pages of equal scales keep their codes");
  const auto carried = download<float>(ctx, moved);
  expect(carried[0] == received[0] && carried[kKeep - 1] == received[kLength - 1] &&
           carried[kKeep] == -1.0f,
         "weights move along");

  const std::size_t size = 1000;
  HipBuffer logprob = upload(ctx, std::vector<float>(2)), entropy = upload(ctx, std::vector<float>(2));
  HipBuffer rank = upload(ctx, std::vector<std::int32_t>(2)), top = upload(ctx, std::vector<std::int32_t>(6));
  s = ctx.token_logprobs_f32(upload(ctx, std::vector<float>(2 * size, 0.5f)), 2, size, size, none,
                             upload(ctx, std::vector<std::int32_t>{0, 700}), 3, logprob, rank,
                             entropy, top, none);
  expect(s.is_ok(), "log probabilities run", s);
  const auto p = download<float>(ctx, logprob), e = download<float>(ctx, entropy);
  const auto r = download<std::int32_t>(ctx, rank), t = download<std::int32_t>(ctx, top);
  expect(std::fabs(p[1] + std::log((double)size)) < 1e-5 && p[0] == p[1] &&
           std::fabs(e[0] - std::log((double)size)) < 1e-5,
         "equal logits share alike");
  expect(r[0] == 0 && r[1] == 700 && t[3] == 0 && t[4] == 1 && t[5] == 2,
         "equal logits stand by index");
  return failures;
}

}  // namespace

int main(int argc, char** argv) {
  const std::string mode = argc > 1 ? argv[1] : "cpu";
  const int failed = mode == "gpu" ? run_gpu() : run_cpu();
  std::printf(failed == 0 ? "all checks passed\n" : "%d checks failed\n", failed);
  return failed == 0 ? 0 : 1;
}
