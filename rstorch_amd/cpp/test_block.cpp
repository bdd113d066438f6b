// The residual block's layers of the C++ mirror: values small enough to check by hand, the state machine,
// and a block against its layers called one by one.
#include <cmath>
#include <cstdio>
#include <vector>

#include "rstorch.hpp"

using namespace rstorch;

static int failures = 0;
#define EXPECT(cond)                                                        \
  do {                                                                      \
    if (!(cond)) { std::printf("FAILED %s:%d  %s\n", __FILE__, __LINE__, #cond); ++failures; } \
  } while (0)

static bool near(const Array2& a, const Array2& b, double tol = 1e-12) {
  if (!a.same_shape(b)) return false;
  auto x = a.to_host(), y = b.to_host();
  for (size_t i = 0; i < x.size(); ++i)
    if (!(std::fabs(x[i] - y[i]) <= tol)) return false;
  return true;
}

template <class F> static bool panics(F f, int status) {
  try { f(); } catch (const Panic& p) { return p.status == status; }
  return false;
}

struct Fixed : InitParameters {
  uint64_t stream;
  explicit Fixed(uint64_t s) : stream(s) {}
  Array2 weight(size_t in, size_t out) const override { return Array2::normal(out, in, 3, stream, 0.0, 1.0 / std::sqrt(double(in))); }
  Array2 bias(size_t, size_t out) const override { return Array2::normal(1, out, 3, stream + 100, 0.0, 0.1); }
};

int main() {
  try {
    {  // a row of +-1 around 5: mean 5, variance 1
      LayerNorm m(4, 0.0);
      EXPECT(near(m.forward(Array2{{4.0, 6.0, 4.0, 6.0}, {10.0, 10.0, 20.0, 20.0}}), Array2{{-1.0, 1.0, -1.0, 1.0}, {-1.0, -1.0, 1.0, 1.0}}));
      EXPECT(panics([&] { m.parameters(); }, RST_ERR_STATE));
      EXPECT(panics([&] { m.backward(Array2::ones(2, 3)); }, RST_ERR_SHAPE));
      // a constant gradient has nothing left once its mean is gone; the bias gradient is its mean over the rows
      EXPECT(near(m.backward(Array2::ones(2, 4)), Array2::zeros(2, 4)));
      EXPECT(near(m.grad_bias(), Array2::ones(1, 4)) && near(m.grad_weight(), Array2{{-1.0, 0.0, 0.0, 1.0}}));
      EXPECT(m.parameters().size() == 2);
      EXPECT(panics([&] { m.backward(Array2::ones(2, 4)); }, RST_ERR_STATE));
      EXPECT(panics([&] { m.forward(Array2::ones(2, 3)); }, RST_ERR_SHAPE));
    }
    {  // dropout: kept values are doubled, the same ones come back in the backward pass, evaluation changes nothing
      Dropout m(0.5, 42);
      Array2 x = Array2::full(30, 30, 3.0);
      auto y = m.forward(x).to_host();
      auto g = m.backward(Array2::ones(30, 30)).to_host();
      size_t kept = 0;
      for (size_t i = 0; i < y.size(); ++i) {
        EXPECT((y[i] == 0.0 && g[i] == 0.0) || (y[i] == 6.0 && g[i] == 2.0));
        kept += y[i] != 0.0;
      }
      EXPECT(kept > 350 && kept < 550);  // 450 +- 6.7 standard deviations
      EXPECT(m.forward(x).to_host() != y);  // the next call draws other numbers
      m.eval();
      EXPECT(near(m.forward(x), x, 0.0) && near(m.backward(x), x, 0.0));
      EXPECT(panics([&] { m.backward(x); }, RST_ERR_STATE));
      EXPECT(panics([&] { Dropout bad(1.0); }, RST_ERR_INVALID_ARGUMENT));
    }
    {  // activations at points with known values
      GELU gelu;
      EXPECT(near(gelu.forward(Array2{{0.0, 1.0, -1.0}}), Array2{{0.0, 0.84134474606854294859, -0.15865525393145705141}}, 1e-15));
      EXPECT(near(gelu.backward(Array2{{2.0, 0.0, 0.0}}), Array2{{1.0, 0.0, 0.0}}, 1e-15));
      EXPECT(panics([&] { gelu.backward(Array2{{1.0, 1.0, 1.0}}); }, RST_ERR_STATE));
      SiLU silu;
      EXPECT(near(silu.forward(Array2{{0.0, std::log(3.0)}}), Array2{{0.0, 0.75 * std::log(3.0)}}, 1e-15));
      EXPECT(near(silu.backward(Array2{{1.0, 0.0}}), Array2{{0.5, 0.0}}, 1e-15));
    }
    {  // a block equals its layers one by one, forward, backward and after a step
      Sequential inner;
      inner.push(LayerNorm(20));
      inner.push(Linear(20, 48, Fixed(1)));
      inner.push(GELU());
      inner.push(Identity());
      inner.push(Linear(48, 20, Fixed(2)));
      Residual block(std::move(inner));
      LayerNorm norm(20);
      Linear first(20, 48, Fixed(1)), second(48, 20, Fixed(2));
      GELU gelu;
      SGD optim(0.1);
      for (int step = 0; step < 3; ++step) {
        Array2 x = Array2::normal(13, 20, 9, step, 0.0, 1.0), g = Array2::normal(13, 20, 9, 50 + step, 0.0, 1.0);
        Array2 want = detail::add(second.forward(gelu.forward(first.forward(norm.forward(x)))), x);
        EXPECT(near(block.forward(x), want));
        Array2 want_g = detail::add(norm.backward(first.backward(gelu.backward(second.backward(g)))), g);
        EXPECT(near(block.backward(g), want_g));
        auto params = block.parameters();
        EXPECT(params.size() == 6);
        EXPECT(near(*params.iter()[0].grad, norm.grad_weight()) && near(*params.iter()[3].grad, first.grad_bias()) &&
               near(*params.iter()[4].grad, second.grad_weight()));
        optim.step(block);
        optim.step(norm);
        optim.step(first);
        optim.step(second);
        EXPECT(near(*block.parameters().iter()[2].parm, first.weight()));
      }
      EXPECT(panics([&] { block.backward(Array2::ones(13, 20)); }, RST_ERR_STATE));
      EXPECT(block.debug() == "Residual(Sequential { layers: [LayerNorm(20), Linear(20, 48), GELU, Identity, Linear(48, 20)] })");
    }
    {  // ReLU and activations on either end of a Linear with the residual in its epilogue
      Residual a(sequential(ReLU(), Linear(6, 6, Fixed(5)), ReLU())), b(sequential(SiLU(), Linear(6, 6, Fixed(5)), SiLU()));
      ReLU r1, r2;
      SiLU s1, s2;
      Linear l(6, 6, Fixed(5));
      Array2 x = Array2::normal(9, 6, 1, 1, 0.0, 1.0), g = Array2::normal(9, 6, 1, 2, 0.0, 1.0);
      EXPECT(near(a.forward(x), detail::add(r2.forward(l.forward(r1.forward(x))), x)));
      EXPECT(near(a.backward(g), detail::add(r1.backward(l.backward(r2.backward(g))), g)));
      EXPECT(near(b.forward(x), detail::add(s2.forward(l.forward(s1.forward(x))), x)));
      EXPECT(near(b.backward(g), detail::add(s1.backward(l.backward(s2.backward(g))), g)));
      EXPECT(panics([&] { Residual(sequential(Linear(6, 7, Fixed(5)))).forward(x); }, RST_ERR_SHAPE));
    }
  } catch (const Panic& p) {
    std::printf("unexpected panic: %s\n", p.what());
    return 1;
  }
  if (failures == 0) std::printf("all block tests passed\n");
  return failures ? 1 : 0;
}
