// GPU tests of the block-scaled launchers of the C++ host surface, on values whose results are known in closed form.
#include <cutile/cutile.hpp>

#include "check.hpp"

using namespace cutile;

static std::shared_ptr<Stream> new_stream() { return Device::create(0).unwrap()->new_stream().unwrap(); }
template <class T>
static Tensor<T> empty(const std::shared_ptr<Stream>& stream, std::vector<int32_t> shape) { return api::Uninitialized<T>(std::move(shape)).sync_on(stream).unwrap(); }

// 24 = 1.5 * 2^4: e4m3 1.5 * 2^8 with scale 2^-4, e2m1 6 with scale 2^2, and in nvfp4 6 with scale 4
TEST(quantise_and_read_back) {
  auto stream = new_stream();
  auto x = api::full<f16>(24.0, {5, 64}).sync_on(stream).unwrap();
  auto back = api::zeros<f16>({5, 64}).sync_on(stream).unwrap();
  auto expect = [&] {
    for (f16 v : api::to_host_vec(back).sync_on(stream).unwrap()) CHECK(f32_from_f16(v) == 24.0f);
    back = api::zeros<f16>({5, 64}).sync_on(stream).unwrap();
  };
  auto d8 = empty<f8e4m3fn>(stream, {5, 64});
  auto s8 = empty<f8e8m0fnu>(stream, {5, 2});
  CHECK(block_quantize(&x, d8.partition_mut({1, 64}), s8.partition_mut({1, 2})).sync_on(stream).is_ok());
  for (auto v : api::to_host_vec(s8).sync_on(stream).unwrap()) CHECK(v.bits == 127 - 4);
  for (auto v : api::to_host_vec(d8).sync_on(stream).unwrap()) CHECK(v.bits == (15 << 3 | 4));
  CHECK(block_dequantize(&d8, &s8, 1.0f, back.partition_mut({1, 64})).sync_on(stream).is_ok());
  expect();
  auto d4 = empty<f4e2m1fnx2>(stream, {5, 32});
  CHECK(block_quantize(&x, d4.partition_mut({1, 32}), s8.partition_mut({1, 2})).generics({"64"}).sync_on(stream).is_ok());
  for (auto v : api::to_host_vec(s8).sync_on(stream).unwrap()) CHECK(v.bits == 127 + 2);
  for (auto v : api::to_host_vec(d4).sync_on(stream).unwrap()) CHECK(v.bits == 0x77);
  CHECK(block_dequantize(&d4, &s8, 1.0f, back.partition_mut({1, 64})).sync_on(stream).is_ok());
  expect();
  auto sn = empty<f8e4m3fn>(stream, {5, 4});
  CHECK(block_quantize(&x, d4.partition_mut({1, 32}), sn.partition_mut({1, 4}), 2.0f).sync_on(stream).is_ok());
  for (auto v : api::to_host_vec(sn).sync_on(stream).unwrap()) CHECK(v.bits == (8 << 3));   // 2
  CHECK(block_dequantize(&d4, &sn, 2.0f, back.partition_mut({1, 64})).sync_on(stream).is_ok());
  expect();
  CHECK(block_quantize(&x, d4.partition_mut({1, 32}), sn.partition_mut({1, 4}), 0.0f).sync_on(stream).is_err());
  CHECK(block_quantize(&x, d8.partition_mut({1, 64}), sn.partition_mut({1, 4})).sync_on(stream).is_err());
}

// rows of 3: the norm is 3 / 3 * w = 2, quantised, and multiplied with themselves: 128 * 2 * 2
TEST(norm_and_activation_in_front_of_the_product) {
  auto stream = new_stream();
  auto r = api::full<bf16>(1.0, {16, 128}).sync_on(stream).unwrap();
  auto x = api::full<bf16>(2.0, {16, 128}).sync_on(stream).unwrap();
  auto w = api::full<bf16>(2.0, {128}).sync_on(stream).unwrap();
  auto sum = api::zeros<bf16>({16, 128}).sync_on(stream).unwrap();
  auto d = empty<f4e2m1fnx2>(stream, {16, 64});
  auto s = empty<f8e8m0fnu>(stream, {16, 4});
  auto product = [&] {
    auto z = partition_op(api::zeros<float>({16, 16}), {128, 128});
    auto res = linear_tile(std::move(z), &d, &d, &s, &s, 0.5f).generics({"128", "128", "128", "64", "4"}).sync_on(stream).unwrap();
    return api::to_host_vec(std::move(std::get<0>(res)).unpartition()).sync_on(stream).unwrap();
  };
  CHECK(add_rms_norm_quantize(&r, &x, &w, d.partition_mut({1, 64}), s.partition_mut({1, 4}), sum.partition_mut({1, 128}), 0.0f).sync_on(stream).is_ok());
  for (bf16 v : api::to_host_vec(sum).sync_on(stream).unwrap()) CHECK(f32_from_bf16(v) == 3.0f);
  for (float v : product()) CHECK(v == 256.0f);
  CHECK(rms_norm_quantize(&x, &w, d.partition_mut({1, 64}), s.partition_mut({1, 4}), 0.0f).sync_on(stream).is_ok());
  for (float v : product()) CHECK(v == 256.0f);
  auto gate = api::full<bf16>(64.0, {16, 128}).sync_on(stream).unwrap();   // silu(64) = 64 in f32
  CHECK(silu_mul_quantize(&gate, &x, d.partition_mut({1, 64}), s.partition_mut({1, 4})).sync_on(stream).is_ok());
  for (float v : product()) CHECK(v == 0.5f * 128 * 128 * 128);
}

int main(int argc, char** argv) { return run_all_tests(argc, argv); }
