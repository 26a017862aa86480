// A feed-forward sublayer through qsml:: -- y = x + (silu(n wg) * (n wu)) wd with
// n = layer_norm(x) -- and its gradients, against the same formulas in double,
// and the error convention.  F32 throughout: binary32 roundings of sums of at most
// 96 terms of size 1 stay below 1e-4.
#include <QuasarML.h>

#include <cmath>
#include <cstdio>
#include <iostream>
#include <stdexcept>
#include <vector>

using std::vector;
using qsml::TensorPtr;
using M = vector<double>;  // row-major

static int passed = 0, failed = 0;

static void check(const char* name, bool ok) {
    if (ok) {
        ++passed;
    } else {
        ++failed;
        std::cout << "FAIL: " << name << "\n";
    }
}

static M values(size_t n, unsigned seed, double scale) {
    M v(n);
    unsigned s = seed * 2654435761u + 12345u;
    for (auto& x : v) {
        s = s * 1664525u + 1013904223u;
        x = static_cast<float>((static_cast<double>(s >> 8) / (1 << 24) * 2.0 - 1.0) * scale);
    }
    return v;
}

static TensorPtr up(const M& v, const vector<qsml::u32>& shape) {
    vector<float> f(v.begin(), v.end());
    return qsml::from_data(f.data(), shape);
}

static M get(const TensorPtr& t) {
    vector<float> f(t->numel());
    t->download(f.data(), f.size() * sizeof(float));
    return M(f.begin(), f.end());
}

static bool close(const TensorPtr& t, const M& ref) {
    if (!t || t->numel() != ref.size()) return false;
    const M v = get(t);
    for (size_t i = 0; i < v.size(); ++i)
        if (!(std::fabs(v[i] - ref[i]) <= 1e-4 * (1.0 + std::fabs(ref[i])))) return false;
    return true;
}

// a [m, k] b [k, n]; ta, tb: the operand is stored transposed
static M mm(const M& a, const M& b, int m, int k, int n, bool ta = false, bool tb = false) {
    M c(size_t(m) * n, 0.0);
    for (int i = 0; i < m; ++i)
        for (int p = 0; p < k; ++p)
            for (int j = 0; j < n; ++j)
                c[i * n + j] += (ta ? a[p * m + i] : a[i * k + p]) * (tb ? b[j * k + p] : b[p * n + j]);
    return c;
}

int main() {
    const int R = 11, C = 40, F = 96;
    const unsigned r = R, c = C, f = F;
    const double eps = 1e-5f;
    const M x = values(R * C, 1, 1), g = values(C, 2, 1), b = values(C, 3, 0.3), wg = values(C * F, 4, 0.2),
            wu = values(C * F, 5, 0.2), wd = values(F * C, 6, 0.2), bd = values(C, 7, 0.5), dy = values(R * C, 8, 1);
    qsml::init();
    auto tx = up(x, {r, c}), tg = up(g, {c}), tb = up(b, {c}), twg = up(wg, {c, f}), twu = up(wu, {c, f}),
         twd = up(wd, {f, c}), tbd = up(bd, {c}), tdy = up(dy, {r, c});

    // forward
    M n(R * C), xh(R * C), rstd(R);
    for (int i = 0; i < R; ++i) {
        double mean = 0, var = 0;
        for (int j = 0; j < C; ++j) mean += x[i * C + j] / C;
        for (int j = 0; j < C; ++j) var += (x[i * C + j] - mean) * (x[i * C + j] - mean) / C;
        rstd[i] = 1.0 / std::sqrt(var + eps);
        for (int j = 0; j < C; ++j) {
            xh[i * C + j] = (x[i * C + j] - mean) * rstd[i];
            n[i * C + j] = xh[i * C + j] * g[j] + b[j];
        }
    }
    const M zg = mm(n, wg, R, C, F), zu = mm(n, wu, R, C, F);
    M h(R * F), a(R * F), da(R * F);
    for (int i = 0; i < R * F; ++i) {
        const double p = 1.0 / (1.0 + std::exp(-zg[i]));
        a[i] = zg[i] * p;
        da[i] = p + zg[i] * p * (1 - p);
        h[i] = a[i] * zu[i];
    }
    M y = mm(h, wd, R, F, C);
    for (int i = 0; i < R * C; ++i) y[i] += x[i] + bd[i % C];

    TensorPtr gate, upk;
    auto tn = qsml::layer_norm(tx, tg, tb);
    auto th = qsml::gated_linear(tn, twg, twu, qsml::Activation::Silu, nullptr, nullptr, &gate, &upk);
    auto ty = qsml::linear(th, twd, tbd, qsml::Activation::None, tx);
    check("gate and up kept", close(gate, zg) && close(upk, zu));
    check("gated_linear", close(th, h));
    check("linear with bias and residual", close(ty, y));

    // backward
    const M dh = mm(dy, wd, R, C, F, false, true), dwd = mm(h, dy, F, R, C, true);
    M dbd(C, 0.0), dg_(R * F), du_(R * F);
    for (int i = 0; i < R * C; ++i) dbd[i % C] += dy[i];
    for (int i = 0; i < R * F; ++i) {
        dg_[i] = dh[i] * zu[i] * da[i];
        du_[i] = dh[i] * a[i];
    }
    M dn = mm(dg_, wg, R, F, C, false, true);
    const M dn2 = mm(du_, wu, R, F, C, false, true);
    for (int i = 0; i < R * C; ++i) dn[i] += dn2[i];
    M dx(R * C), dgam(C, 0.0), dbet(C, 0.0);
    for (int i = 0; i < R; ++i) {
        double c1 = 0, c2 = 0;
        for (int j = 0; j < C; ++j) {
            c1 += dn[i * C + j] * g[j] / C;
            c2 += dn[i * C + j] * g[j] * xh[i * C + j] / C;
        }
        for (int j = 0; j < C; ++j) {
            dx[i * C + j] = rstd[i] * (dn[i * C + j] * g[j] - c1 - xh[i * C + j] * c2);
            dgam[j] += dn[i * C + j] * xh[i * C + j];
            dbet[j] += dn[i * C + j];
        }
    }
    auto gl = qsml::linear_backward(th, twd, qsml::Activation::None, nullptr, tdy, true);
    check("linear_backward", close(gl.dx, dh) && close(gl.dw, dwd) && close(gl.dbias, dbd));
    auto gg = qsml::gated_linear_backward(tn, twg, twu, qsml::Activation::Silu, gate, upk, gl.dx, true);
    check("gated_linear_backward dx", close(gg.dx, dn));
    check("gated_linear_backward dw",
          close(gg.dw_gate, mm(n, dg_, C, R, F, true)) && close(gg.dw_up, mm(n, du_, C, R, F, true)));
    M sg(F, 0.0), su(F, 0.0);
    for (int i = 0; i < R * F; ++i) {
        sg[i % F] += dg_[i];
        su[i % F] += du_[i];
    }
    check("gated_linear_backward db", close(gg.db_gate, sg) && close(gg.db_up, su));
    auto gn = qsml::layer_norm_backward(tx, tg, gg.dx);
    check("layer_norm_backward", close(gn.dx, dx) && close(gn.dgamma, dgam) && close(gn.dbeta, dbet));

    // a transposed weight is read in place; three dims fold; an activation's backward pass
    auto wt = qsml::transpose(up(M([&] {
        M t(F * C);
        for (int i = 0; i < F; ++i)
            for (int j = 0; j < C; ++j) t[j * F + i] = wd[i * C + j];
        return t;
    }()), {c, f}));
    check("transposed weight", close(qsml::linear(th, wt, tbd, qsml::Activation::None, tx), y));
    TensorPtr pre;
    auto x3 = qsml::reshape(tx, {1, r, c});
    auto relu = qsml::linear(x3, twg, nullptr, qsml::Activation::Relu, nullptr, &pre);
    check("three dims", relu->rank() == 3 && relu->dim(2) == f && pre->rank() == 3);
    const M z = mm(x, wg, R, C, F), ones(R * F, 1.0);
    M zr = z, dz(R * F);
    for (int i = 0; i < R * F; ++i) {
        zr[i] = z[i] > 0 ? z[i] : 0;
        dz[i] = z[i] > 0 ? 1 : 0;
    }
    check("relu layer", close(relu, zr));
    auto gr = qsml::linear_backward(x3, twg, qsml::Activation::Relu, pre, up(ones, {1, r, f}));
    check("relu layer's gradients", close(gr.dx, mm(dz, wg, R, F, C, false, true)) &&
                                        close(gr.dw, mm(x, dz, C, R, F, true)) && !gr.dbias);
    // errors
    auto throws = [](auto fn) {
        try {
            fn();
        } catch (const std::runtime_error&) {
            return true;
        }
        return false;
    };
    check("inner dims differ", throws([&] { qsml::linear(tx, twd); }));
    check("pre needed", throws([&] { qsml::linear_backward(tx, twg, qsml::Activation::Gelu, nullptr, gate); }));
    check("gamma's size", throws([&] { qsml::layer_norm_backward(tx, tbd->view({1, c}), up(values(R, 9, 1), {r})); }));
    check("null weight", throws([&] { qsml::gated_linear(tx, twg, nullptr); }));
    check("usable after errors", close(qsml::linear(th, twd, tbd, qsml::Activation::None, tx), y));
    qsml::shutdown();
    std::cout << "passed " << passed << " failed " << failed << "\n";
    return failed ? 1 : 0;
}
