// The sequence operators through the C++ host layer: values that can be written down by hand, states carried from a prompt to
// single tokens, gradients by differences, refusals. Exit code 0 = every check passed. Needs an MI355X; run by
// tests/test_sequence_gpu.py.
#include <cmath>
#include <cstdio>
#include <stdexcept>
#include <vector>

#include "am_hip_tensor.hpp"

using am::HipTensor;
using am::Shape;
using am::toHip;

static int g_failed = 0, g_checked = 0;
#define CHECK(cond)                                                          \
  do {                                                                       \
    ++g_checked;                                                             \
    if (!(cond)) { ++g_failed; std::printf("FAILED %s:%d  %s\n", __FILE__, __LINE__, #cond); } \
  } while (0)
#define EXPECT_THROW(expr, EXC)                                              \
  do {                                                                       \
    ++g_checked;                                                             \
    bool ok_ = false;                                                        \
    try { (void)(expr); } catch (const EXC&) { ok_ = true; } catch (...) {}  \
    if (!ok_) { ++g_failed; std::printf("FAILED %s:%d  %s did not throw %s\n", __FILE__, __LINE__, #expr, #EXC); } \
  } while (0)

template <typename T> static bool near(const HipTensor<T>& t, const std::vector<double>& want, double tol) {
  const auto got = t.toCpu();
  if (got.size() != want.size()) return false;
  for (size_t i = 0; i < got.size(); ++i)
    if (!(std::fabs((double)got[i] - want[i]) <= tol)) return false;
  return true;
}
static std::vector<double> numbers(size_t n, unsigned seed) {
  std::vector<double> v(n);
  unsigned s = seed;
  for (auto& x : v) { s = s * 1664525u + 1013904223u; x = (double)(s >> 8) / (1 << 24) * 2 - 1; }
  return v;
}
template <typename T> static HipTensor<T> dev(const std::vector<double>& v, const Shape& s) { return toHip<T>(std::vector<T>(v.begin(), v.end()), s); }
static double dot(const std::vector<double>& a, const std::vector<double>& b) {
  double s = 0;
  for (size_t i = 0; i < a.size(); ++i) s += a[i] * b[i];
  return s;
}

template <typename T> static void rotary_quarters() {
  // a quarter turn a position: (1, 2) -> (-2, 1) -> (-1, -2), the element behind the pair stays
  const double quarter = std::acos(0.0), u = sizeof(T) == 4 ? 1e-6 : 1e-14;
  auto x = dev<T>({1, 2, 7, 1, 2, 7, 1, 2, 7}, {1, 3, 1, 3});
  auto f = toHip<double>({quarter}, {1});
  CHECK(near(am::rotary<T>(x, nullptr, f), {1, 2, 7, -2, 1, 7, -1, -2, 7}, u));
  auto at = toHip<int64_t>({1, 1, -1}, {1, 3});
  CHECK(near(am::rotary<T>(x, &at, f, AM_ROTARY_INTERLEAVED, T(2)), {-4, 2, 7, -4, 2, 7, 4, -2, 7}, u));
  CHECK(near(am::rotary_backward<T>(am::rotary<T>(x, &at, f), &at, f), {1, 2, 7, 1, 2, 7, 1, 2, 7}, u));
  EXPECT_THROW(am::rotary<T>(x, &at, toHip<double>({1, 2}, {2})), std::invalid_argument);
}

template <typename T> static void attention_by_hand() {
  // one head of 1 x 1, decay 1/2: the state is 1, 1/2 + 2, 5/4 + 3
  auto q = dev<T>({1, 10, 100}, {1, 3, 1, 1}), k = dev<T>({1, 1, 1}, {1, 3, 1, 1}), v = dev<T>({1, 2, 3}, {1, 3, 1, 1});
  auto g = dev<T>({std::log(0.5)}, {1});
  HipTensor<T> last;
  CHECK(near(am::decay_attention<T>(q, k, v, g, T(1), nullptr, &last), {1, 25, 425}, 1e-4));
  CHECK(near(last, {4.25}, 1e-6));
  auto len = toHip<int64_t>({2}, {1});
  CHECK(near(am::decay_attention<T>(q, k, v, g, T(2), nullptr, &last, &len), {2, 50, 0}, 1e-4) && near(last, {2.5}, 1e-6));
  // the next token continues
  auto o = am::decay_attention_step<T>(dev<T>({100}, {1, 1, 1}), dev<T>({1}, {1, 1, 1}), dev<T>({3}, {1, 1, 1}), g, last);
  CHECK(near(o, {425}, 1e-4) && near(last, {4.25}, 1e-6));
  EXPECT_THROW(am::decay_attention<T>(q, k, dev<T>({1, 2}, {1, 2, 1, 1}), g), std::invalid_argument);
  EXPECT_THROW(am::decay_attention<T>(q, k, v, dev<T>({1, 2}, {2})), std::invalid_argument);
}

static void attention_gradients() {
  const Shape qs{1, 40, 2, 5}, ks{1, 40, 1, 5}, vs{1, 40, 1, 3}, os{1, 40, 2, 3}, ss{1, 2, 5, 3};
  const auto q = numbers(400, 1), k = numbers(200, 2), v = numbers(120, 3), go = numbers(240, 4), s = numbers(30, 5), gs = numbers(30, 6);
  auto g = toHip<double>({-0.2, -0.01}, {2});
  auto loss = [&](const std::vector<double>& q_, const std::vector<double>& k_, const std::vector<double>& v_, const std::vector<double>& s_) {
    auto st = dev<double>(s_, ss);
    HipTensor<double> last;
    return dot(am::decay_attention<double>(dev<double>(q_, qs), dev<double>(k_, ks), dev<double>(v_, vs), g, 0.5, &st, &last).toCpu(), go) + dot(last.toCpu(), gs);
  };
  auto st = dev<double>(s, ss), dst = dev<double>(gs, ss);
  auto r = am::decay_attention_backward<double>(dev<double>(go, os), dev<double>(q, qs), dev<double>(k, ks), dev<double>(v, vs), g, 0.5, &st, &dst);
  CHECK(r.size() == 4 && r[0].shape == qs && r[1].shape == ks && r[2].shape == vs && r[3].shape == ss);
  const std::vector<double>* at[4] = {&q, &k, &v, &s};
  for (int i = 0; i < 4; ++i) {
    const auto way = numbers(at[i]->size(), 10 + i);
    const double h = 1e-5;
    double side[2];
    for (int w = 0; w < 2; ++w) {
      std::vector<double> m = *at[i];
      for (size_t e = 0; e < m.size(); ++e) m[e] += (w ? -h : h) * way[e];
      side[w] = loss(i == 0 ? m : q, i == 1 ? m : k, i == 2 ? m : v, i == 3 ? m : s);
    }
    const double want = (side[0] - side[1]) / (2 * h), got = dot(r[i].toCpu(), way);
    CHECK(std::fabs(got - want) <= 1e-7 * (1 + std::fabs(want)));
  }
}

template <typename T> static void norms_by_hand() {
  // two samples of two groups of two channels: (1, 3) -> (-1, 1), (10, 20) -> (-1, 1)
  auto x = dev<T>({1, 3, 10, 20, 5, 5, -2, 2}, {2, 4}), w = dev<T>({1, 2, 1, 1}, {4}), b = dev<T>({0, 0, 1, 0}, {4});
  const double u = sizeof(T) == 4 ? 1e-5 : 1e-12;
  std::vector<HipTensor<T>> kept;
  CHECK(near(am::group_norm<T>(x, &w, &b, 2, T(0.0), AM_ACT_RELU), {0, 2, 0, 1, NAN, NAN, 0, 1}, u) == false);   // 0 / 0 where all are equal and eps is 0
  auto y = am::group_norm<T>(x, &w, &b, 2, T(1e-12), AM_ACT_RELU, &kept);
  // eps = 1e-12 beside a variance of 1 scales by 1 / sqrt(1 + 1e-12) = 1 - 5e-13, which takes 1e-12 from the 2
  CHECK(near(y, {0, 2, 0, 1, 0, 0, 0, 1}, u + 1e-12));
  CHECK(near(kept[0], {2, 15, 5, 0}, u));
  // through a permuted view: the same numbers with the channels first
  auto first = dev<T>({1, 3, 10, 20}, {1, 2, 2});
  std::swap(first.strides[1], first.strides[2]);
  CHECK(near(am::group_norm<T>(first, nullptr, nullptr, 2, T(1e-12)), {-1, -1, 1, 1}, u));
  auto d = am::group_norm_backward<T>(dev<T>({1, 1, 1, 1, 1, 1, 1, 1}, {2, 4}), x, nullptr, nullptr, kept, 2);
  CHECK(near(d[0], {0, 0, 0, 0, 0, 0, 0, 0}, 1e-3 * u + (sizeof(T) == 4 ? 1e-6 : 0)) && d[1].shape.empty() && d[2].shape.empty());   // a shift of a group changes nothing
  EXPECT_THROW(am::group_norm<T>(x, &w, &b, 3), std::invalid_argument);
  auto three = dev<T>({1, 2, 3}, {3});
  EXPECT_THROW(am::group_norm<T>(x, &three, &b, 2), std::invalid_argument);
}

int main() {
  try {
    rotary_quarters<float>();
    rotary_quarters<double>();
    attention_by_hand<float>();
    attention_by_hand<double>();
    attention_gradients();
    norms_by_hand<float>();
    norms_by_hand<double>();
    am::sync();
  } catch (const std::exception& e) {
    std::printf("unexpected exception: %s\n", e.what());
    return 2;
  }
  std::printf("%d checks, %d failed\n", g_checked, g_failed);
  return g_failed ? 1 : 0;
}
