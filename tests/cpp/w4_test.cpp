// w4_test.cpp -- the C++ layer's 4-bit weights: sizes and views (no device), and a Linear that is
// recorded over them.
#include <cmath>
#include <vector>

#include "ammon/ammon.hpp"
#include "check.hpp"

using ammon::DType;
using ammon::Shape;
using ammon::Tensor;
using ammon::TensorView;

namespace {
template <typename F> bool throws(F &&f) {
  try {
    f();
  } catch (const ammon::Error &e) {
    return e.status() == AMMON_E_VALIDATION;
  }
  return false;
}
}  // namespace

TEST(storage_bytes_of_w4) {
  CHECK(ammon::storage_bytes(Shape::matrix(16, 128), DType::W4) == 1056);
  CHECK(ammon::storage_bytes(Shape::matrix(17, 129), DType::W4) == 4 * 1056);
  CHECK(ammon::storage_bytes(Shape::from_dims({3, 17, 129}), DType::W4) == 12 * 1056);
  CHECK(throws([] { ammon::storage_bytes(Shape::vector(128), DType::W4); }));
  CHECK(throws([] { ammon::dtype_size(DType::W4); }));
}

TEST(views_of_w4) {
  char *base = (char *)4096;
  const TensorView v(base, Shape::from_dims({4, 17, 129}), DType::W4);
  const TensorView l = v.narrow(0, 3, 1);
  CHECK((char *)l.data() == base + 3 * 4 * 1056);
  CHECK(l.reshape({17, 129}).nbytes() == 4 * 1056);
  CHECK(throws([&] { v.narrow(1, 0, 16); }));
  CHECK(throws([&] { v.narrow(2, 0, 128); }));
  CHECK(throws([&] { l.reshape({129, 17}); }));
}

TEST(linear_over_w4) {
  const ammon::Runtime rt = ammon::Runtime::create(0);
  const uint32_t d = 33, n = 130;
  std::vector<float> w(d * n), x(n);
  for (uint32_t i = 0; i < d * n; ++i) w[i] = (float)((i * 7 + i / n) % 15) - 7.f;  // codes of scale 1
  for (uint32_t r = 0; r < d; ++r) w[r * n] = w[r * n + 128] = 7.f;  // (each group reaches 7)
  for (uint32_t i = 0; i < n; ++i) x[i] = (float)(i % 9) - 4.f;
  const Tensor numbers = Tensor::from_f32(rt, Shape::matrix(d, n), w);
  const Tensor w4 = Tensor::zeros(rt, Shape::matrix(d, n), DType::W4);
  ammon::check(ammon_w4_store(rt.raw(), nullptr, numbers.data(), AMMON_F32, d, n, w4.data()));
  const Tensor in = Tensor::from_f32(rt, Shape::vector(n), x);
  const Tensor out = Tensor::zeros(rt, Shape::vector(d), DType::F32);
  ammon_stream_synchronize(rt.raw(), nullptr);
  ammon::Scheme s(rt);
  ammon::Linear(rt).record(s, w4.view(), in.view(), out.view());
  s.submit();
  s.synchronize();
  const std::vector<float> got = out.to_f32();
  for (uint32_t r = 0; r < d; ++r) {
    float want = 0.f;  // whole numbers: exact
    for (uint32_t i = 0; i < n; ++i) want += w[r * n + i] * x[i];
    CHECK(got[r] == want);
  }
  // a table of 4-bit rows is not gathered from
  const Tensor step = ammon::DecodeStep::parcel(rt);
  const size_t before = s.ir_node_count();
  CHECK(throws([&] { ammon::kernels::embed(s, "embed", w4.view(), step, in.view()); }));
  CHECK(s.ir_node_count() == before);
}

int main(int argc, char **argv) { return check::run_all(argc, argv); }
