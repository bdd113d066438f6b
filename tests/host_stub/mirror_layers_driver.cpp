// The C++ mirror's layer lists over hip_stub.cpp: a subclass of a layer that overrides forward and backward is called
// wherever it stands in a Sequential or a Residual, in its own place, and the layers themselves stay joined.  Kernels do
// not run; what is counted is calls and launches.
#include <cstdio>
#include <cstdlib>

#include "../../rstorch_amd/cpp/rstorch.hpp"

using namespace rstorch;

extern "C" long hip_stub_launch_count();

static int g_forward = 0, g_backward = 0;
static long g_launches_at_forward = 0;  // when the overridden forward ran

template <class Base>
struct Own : Base {
  using Base::Base;
  Array2 forward(Array2 input) override {
    ++g_forward;
    g_launches_at_forward = hip_stub_launch_count();
    return Base::forward(std::move(input));
  }
  Array2 backward(Array2 gradient) override {
    ++g_backward;
    return Base::backward(std::move(gradient));
  }
};

#define REQUIRE(cond)                                                                    \
  do {                                                                                   \
    if (!(cond)) {                                                                       \
      std::fprintf(stderr, "%s:%d: %s (%s)\n", __FILE__, __LINE__, #cond, g_case);       \
      std::exit(1);                                                                      \
    }                                                                                    \
  } while (0)
static const char* g_case = "";

static Array2 array() { return Array2::zeros(4, 6); }
static Linear linear() { return Linear(6, 6); }

template <class Model>
static void once(Model&& model) {
  g_forward = g_backward = 0;
  (void)model.forward(array());
  REQUIRE(g_forward == 1);
  (void)model.backward(array());
  REQUIRE(g_backward == 1);
}

// `make` builds the overridden layer; it stands behind, in front of, between
template <class Make>
static void everywhere(const char* name, Make make) {
  g_case = name;
  once(sequential(linear(), make()));
  once(sequential(make(), linear()));
  once(sequential(linear(), make(), linear()));
  once(sequential(linear(), make(), GELU()));
  once(sequential(SiLU(), make(), linear()));
  once(Residual(sequential(linear(), make())));
  once(Residual(sequential(make(), linear())));
  once(Residual(sequential(linear(), make(), linear())));
  once(Residual(sequential(linear(), make(), GELU())));
  once(Residual(sequential(SiLU(), make(), linear())));
}

template <class Model>
static long launches(Model&& model, bool backward) {
  const long before = hip_stub_launch_count();
  Array2 out = model.forward(array());
  const long forward = hip_stub_launch_count() - before;
  if (!backward) return forward;
  (void)model.backward(array()).data();
  return hip_stub_launch_count() - before - forward;
}

int main() {
  everywhere("GELU", [] { return Own<GELU>(); });
  everywhere("SiLU", [] { return Own<SiLU>(); });
  everywhere("ReLU", [] { return Own<ReLU>(); });
  everywhere("Identity", [] { return Own<Identity>(); });
  everywhere("Dropout", [] { return Own<Dropout>(0.5); });
  everywhere("LayerNorm", [] { return Own<LayerNorm>(size_t(6)); });
  everywhere("Linear", [] { return Own<Linear>(size_t(6), size_t(6)); });
  g_case = "Identity between a Linear and its activation";
  for (int kind = 0; kind < 2; ++kind) {
    Sequential m;
    m.push(linear());
    m.push(Own<Identity>());
    if (kind == 0) m.push(GELU());
    else m.push(ReLU());
    Array2 x = array();
    const long before = hip_stub_launch_count();
    (void)m.forward(x);
    REQUIRE(g_launches_at_forward == before + 1);            // the product alone lies in front of it
    REQUIRE(hip_stub_launch_count() == before + 2);          // and the activation behind it
  }
  g_case = "the layers themselves";
  // one launch more for the rows' zeros of array()
  REQUIRE(launches(Residual(sequential(linear(), GELU())), false) == 2);
  REQUIRE(launches(sequential(linear(), SiLU()), false) == 2);
  REQUIRE(launches(sequential(linear(), Identity(), GELU()), false) == 2);
  REQUIRE(launches(Residual(sequential(linear(), ReLU())), false) == 2);
  REQUIRE(launches(Residual(sequential(linear(), Dropout(0.5))), false) == 3);
  REQUIRE(launches(Residual(sequential(linear(), GELU(), linear())), true) ==
          launches(sequential(linear(), GELU(), linear()), true));
  std::printf("mirror layers ok\n");
  return 0;
}
