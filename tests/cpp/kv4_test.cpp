// kv4_test.cpp -- the C++ layer's 4-bit KV cache: sizes and views (no device), and
// a KvCache with the recorders that write and read it.
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

TEST(storage_bytes_of_kv4) {
  CHECK(ammon::storage_bytes(Shape::from_dims({3, 7, 128}), DType::KV4) == 3 * 7 * 80);
  CHECK(ammon::storage_bytes(Shape::from_dims({2, 5, 3, 7, 33}), DType::KV4) == 10 * (3 * 7 * 40 + 8));
  CHECK(ammon::storage_bytes(Shape::from_dims({3, 7, 128}), DType::BF16) == 3 * 7 * 256);
  CHECK(throws([] { ammon::storage_bytes(Shape::from_dims({7, 128}), DType::KV4); }));
  CHECK(throws([] { ammon::dtype_size(DType::KV4); }));
}

TEST(views_of_kv4) {
  char *base = (char *)4096;
  const TensorView v(base, Shape::from_dims({4, 2, 16, 64}), DType::KV4);
  const TensorView l = v.narrow(0, 3, 1);
  CHECK((char *)l.data() == base + 3 * 2 * 16 * 40);
  CHECK(l.reshape({2, 16, 64}).nbytes() == 2 * 16 * 40);
  CHECK(throws([&] { v.narrow(1, 0, 1); }));
  CHECK(throws([&] { v.narrow(2, 0, 4); }));
  CHECK(throws([&] { l.reshape({16, 2, 64}); }));
  CHECK(throws([&] { l.reshape({2, 8, 128}); }));
}

TEST(stacked_caches_are_aligned) {
  // 3 x 7 rows of 40 bytes are no multiple of 16
  const TensorView v((char *)4096, Shape::from_dims({2, 5, 3, 7, 33}), DType::KV4);
  const TensorView a = v.narrow(0, 1, 1).narrow(1, 3, 1);
  CHECK((char *)a.data() == (char *)4096 + 8 * 848);
  CHECK(a.reshape({3, 7, 33}).nbytes() == 840);
  CHECK(v.nbytes() == 10 * 848);
}

TEST(cache_records_and_reads_back) {
  const ammon::Runtime rt = ammon::Runtime::create(0);
  const uint32_t kv = 2, head = 64, seq = 16;
  ammon::KvCache cache(rt, 3, seq, kv, head, DType::KV4);
  ammon::KvLayer layer = cache.layer(1);
  CHECK(layer.key.nbytes() == kv * seq * 40);
  std::vector<float> rows(kv * head);
  for (size_t i = 0; i < rows.size(); ++i) rows[i] = (float)(i % 16) - 3.f;  // 16 values: exact
  const Tensor src = Tensor::from_f32(rt, Shape::vector(kv * head), rows);
  const Tensor step = ammon::DecodeStep::parcel(rt);
  ammon::DecodeStep::deposit(rt, step, {0, 5});
  ammon::Scheme s(rt);
  ammon::kernels::cache_store(s, "store", src.view(), layer.value, step);
  ammon_stream_synchronize(rt.raw(), nullptr);
  s.submit();
  s.synchronize();
  const std::vector<uint8_t> bytes = cache.layer_to_host_reference_order(1, true);
  const float *got = (const float *)bytes.data();
  for (uint32_t t = 0; t < seq; ++t)
    for (uint32_t i = 0; i < kv * head; ++i)
      CHECK(got[t * kv * head + i] == (t == 5 ? rows[i] : 0.f));
  const std::vector<uint8_t> other = cache.layer_to_host_reference_order(2, true);
  for (size_t i = 0; i < other.size(); ++i) CHECK(other[i] == 0);
  // an in-place rotation of quantised rows is refused when it is recorded
  const Tensor q = Tensor::zeros(rt, Shape::from_dims({4, head}), DType::F32);
  const auto table = ammon::kernels::rope_table(rt, 10000.f, head, seq);
  const TensorView tv = table->view().reshape({seq, head / 2, 2});
  const size_t before = s.ir_node_count();
  CHECK(throws([&] { ammon::kernels::rope(s, "rope", q.view(), layer.key, step, tv); }));
  CHECK(s.ir_node_count() == before);
}

int main(int argc, char **argv) { return check::run_all(argc, argv); }
