// GPU tests of the paged cache's launchers and of adjusted logits on the C++ host surface, on values whose results are known in closed form.
#include <cutile/cutile.hpp>

#include "check.hpp"

using namespace cutile;

static std::shared_ptr<Stream> new_stream() { return Device::create(0).unwrap()->new_stream().unwrap(); }
template <class T>
static Tensor<T> on_device(const std::shared_ptr<Stream>& stream, std::vector<T> v, std::vector<int32_t> shape) {
  return reshape_op(api::copy_host_vec_to_device(std::make_shared<std::vector<T>>(std::move(v))), std::move(shape)).sync_on(stream).unwrap();
}

// Two sequences of 3 and 1 tokens on pages of 2 tokens: keys of zeros weigh all tokens alike, so attention gives the one value that there is.
TEST(a_step_over_a_paged_cache) {
  auto stream = new_stream();
  auto table = on_device<int32_t>(stream, {4, 1, 2, -1}, {2, 2});
  auto starts = on_device<int32_t>(stream, {0, 3, 4}, {3});
  auto lens = on_device<int32_t>(stream, {3, 1}, {2});
  auto nk = api::zeros<f16>({4, 2, 64}).sync_on(stream).unwrap();
  auto nv = api::full<f16>(24.0, {4, 2, 64}).sync_on(stream).unwrap();
  auto q = api::full<f16>(3.0, {4, 6, 64}).sync_on(stream).unwrap();
  auto expect = [&](Tensor<f16>& t, float value) {
    for (f16 v : api::to_host_vec(t).sync_on(stream).unwrap()) CHECK(f32_from_f16(v) == value);
  };
  auto out = api::zeros<f16>({4, 6, 64}).sync_on(stream).unwrap();
  auto rk = api::full<f16>(1.0, {4, 2, 64}).sync_on(stream).unwrap(), rv = api::zeros<f16>({4, 2, 64}).sync_on(stream).unwrap();
  {
    auto k = api::full<f16>(7.0, {5, 2, 2, 64}).sync_on(stream).unwrap(), v = api::full<f16>(7.0, {5, 2, 2, 64}).sync_on(stream).unwrap();
    CHECK(paged_cache_write(&nk, &nv, &k, &v, &table, &starts, &lens).sync_on(stream).is_ok());
    CHECK(paged_cache_read(&k, &v, &table, &starts, &lens, rk.partition_mut({1, 2, 64}), rv.partition_mut({1, 2, 64})).sync_on(stream).is_ok());
    expect(rk, 0.0f), expect(rv, 24.0f);
    CHECK(paged_attention(&q, &k, &v, &table, &starts, &lens, out.partition_mut({1, 6, 64}), 0.125f).sync_on(stream).is_ok());
    expect(out, 24.0f);
    CHECK(paged_attention(&q, &k, &v, &table, &starts, &lens, out.partition_mut({1, 6, 64}), 0.125f, -1).sync_on(stream).is_err());
  }
  auto k = api::Uninitialized<f8e4m3fn>({5, 2, 2, 64}).sync_on(stream).unwrap(), v = api::Uninitialized<f8e4m3fn>({5, 2, 2, 64}).sync_on(stream).unwrap();
  auto ks = api::Uninitialized<f8e8m0fnu>({5, 2, 2, 2}).sync_on(stream).unwrap(), vs = api::Uninitialized<f8e8m0fnu>({5, 2, 2, 2}).sync_on(stream).unwrap();
  auto workspace = api::zeros<int32_t>({65536}).sync_on(stream).unwrap();
  CHECK(paged_cache_write(&nk, &nv, &k, &v, &table, &starts, &lens, &ks, &vs).sync_on(stream).is_ok());
  rv = api::zeros<f16>({4, 2, 64}).sync_on(stream).unwrap();
  CHECK(paged_cache_read(&k, &v, &table, &starts, &lens, rk.partition_mut({1, 2, 64}), rv.partition_mut({1, 2, 64}), &ks, &vs).sync_on(stream).is_ok());
  expect(rv, 24.0f);
  out = api::zeros<f16>({4, 6, 64}).sync_on(stream).unwrap();
  CHECK(paged_attention(&q, &k, &v, &table, &starts, &lens, out.partition_mut({1, 6, 64}), 0.125f, 2, 3, 3, &ks, &vs, &workspace).sync_on(stream).is_ok());
  expect(out, 24.0f);
  CHECK(paged_cache_write(&nk, &nv, &k, &v, &table, &starts, &lens).sync_on(stream).is_err());   // an 8-bit cache without scales
}

// 2 with repetition 2 is 1; token 5 stands twice behind the prompt: 1 - 0.25 - 2 * 0.125
TEST(adjusted_logits) {
  auto stream = new_stream();
  auto logits = api::full<float>(2.0f, {1, 40}).sync_on(stream).unwrap();
  auto out = api::zeros<float>({1, 40}).sync_on(stream).unwrap();
  auto tokens = on_device<int32_t>(stream, {9, 5, 5, 7}, {1, 4});
  auto prompt = on_device<int32_t>(stream, {1}, {1}), used = on_device<int32_t>(stream, {3}, {1});
  auto repetition = on_device<float>(stream, {2.0f}, {1}), presence = on_device<float>(stream, {0.25f}, {1}), frequency = on_device<float>(stream, {0.125f}, {1});
  CHECK(adjust_logits(&logits, out.partition_mut({1, 40}), &tokens, &prompt, &used, &repetition, &presence, &frequency).sync_on(stream).is_ok());
  auto host = api::to_host_vec(out).sync_on(stream).unwrap();
  for (int i = 0; i < 40; ++i) CHECK(host[i] == (i == 5 ? 0.5f : i == 9 ? 1.0f : 2.0f));
  CHECK(adjust_logits(&logits, out.partition_mut({1, 40})).sync_on(stream).is_ok());
  for (float v : api::to_host_vec(out).sync_on(stream).unwrap()) CHECK(v == 2.0f);
  CHECK(adjust_logits(&logits, out.partition_mut({1, 40}), Absent{}, &prompt).sync_on(stream).is_err());
}

int main(int argc, char** argv) { return run_all_tests(argc, argv); }
