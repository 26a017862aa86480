// An attention sublayer through qsml:: -- queries and keys out of one projection, normed and
// rotated, then attention with a window and first tokens -- and its gradients, against the same
// formulas in double; next tokens over a cache; the error convention.  F32 throughout: binary32
// roundings of sums of at most 64 terms of size 1 stay below 1e-4.
#include <QuasarML.h>

#include <cmath>
#include <cstdio>
#include <iostream>
#include <stdexcept>
#include <vector>

using std::vector;
using qsml::TensorPtr;
using M = vector<double>;

static int passed = 0, failed = 0;

static void check(const char* name, bool ok) {
    if (ok) {
        ++passed;
    } else {
        ++failed;
        std::cout << "FAIL: " << name << "\n";
    }
}

static M values(size_t n, unsigned seed, double scale, double mean = 0) {
    M v(n);
    unsigned s = seed * 2654435761u + 12345u;
    for (auto& x : v) {
        s = s * 1664525u + 1013904223u;
        x = static_cast<float>((static_cast<double>(s >> 8) / (1 << 24) * 2.0 - 1.0) * scale + mean);
    }
    return v;
}
static TensorPtr up(const M& v, const vector<qsml::u32>& shape) {
    vector<float> f(v.begin(), v.end());
    return qsml::from_data(f.data(), shape);
}
static TensorPtr ints(const vector<int>& v, const vector<qsml::u32>& shape) {
    return qsml::from_data(v.data(), shape, qsml::DataType::I32);
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

const int B = 2, T = 13, HQ = 4, HK = 2, D = 8, W = 5, SINKS = 2, R = 6;
const double EPS = 1e-6f;

// y = rotated norm of x [B, T, H, D]; with dy: dx and dw.
static M norm_rotary(const M& x, int H, const M& w, const M& freq, const vector<int>& pos, const M* dy = nullptr, M* dw = nullptr) {
    M out(x.size());
    for (int r = 0; r < B * T * H; ++r) {
        const double *a = &x[size_t(r) * D], p = pos[r / H];
        double sq = 0;
        for (int c = 0; c < D; ++c) sq += a[c] * a[c];
        const double s = 1 / std::sqrt(sq / D + EPS);
        M y(D), g(D);
        for (int c = 0; c < D; ++c) y[c] = dy ? (*dy)[size_t(r) * D + c] : a[c] * s * w[c];
        for (int i = 0; i < R / 2; ++i) {
            const double t = p * freq[i] * (dy ? -1 : 1), u = y[i], v = y[R / 2 + i];
            y[i] = u * std::cos(t) - v * std::sin(t);
            y[R / 2 + i] = v * std::cos(t) + u * std::sin(t);
        }
        double along = 0;
        for (int c = 0; c < D; ++c) along += y[c] * w[c] * a[c] * s / D;
        for (int c = 0; c < D; ++c) {
            out[size_t(r) * D + c] = dy ? s * (y[c] * w[c] - a[c] * s * along) : y[c];
            if (dw) (*dw)[c] += y[c] * a[c] * s;
        }
    }
    return out;
}

struct Grads {
    M q, k, v;
};
// o of q over k, v [B, T, ..]; nk: keys of each sequence; with dout: gradients.
static M attend(const M& q, const M& k, const M& v, int nq, const vector<int>& nk, const M* dout = nullptr, Grads* g = nullptr) {
    M o(q.size(), 0.0);
    const double scale = 1 / std::sqrt(double(D));
    for (int b = 0; b < B; ++b)
        for (int h = 0; h < HQ; ++h)
            for (int i = 0; i < nq; ++i) {
                const int p = nk[b] - nq + i, kh = h / (HQ / HK);
                const size_t qi = ((size_t(b) * nq + i) * HQ + h) * D;
                auto at = [&](int j) { return ((size_t(b) * T + j) * HK + kh) * D; };
                M e(T, 0.0), dp(T, 0.0);
                double sum = 0, delta = 0;
                for (int j = 0; j <= p; ++j) {
                    if (p - j >= W && j >= SINKS) continue;
                    double s = 0;
                    for (int c = 0; c < D; ++c) s += q[qi + c] * k[at(j) + c];
                    sum += e[j] = std::exp(s * scale);
                }
                for (int j = 0; j < T; ++j) {
                    e[j] /= sum > 0 ? sum : 1;
                    for (int c = 0; c < D; ++c) o[qi + c] += e[j] * v[at(j) + c];
                    if (dout)
                        for (int c = 0; c < D; ++c) dp[j] += (*dout)[qi + c] * v[at(j) + c];
                    delta += e[j] * dp[j];
                }
                for (int j = 0; j < T && dout; ++j)
                    for (int c = 0; c < D; ++c) {
                        const double ds = e[j] * (dp[j] - delta) * scale;
                        g->q[qi + c] += ds * k[at(j) + c];
                        g->k[at(j) + c] += ds * q[qi + c];
                        g->v[at(j) + c] += e[j] * (*dout)[qi + c];
                    }
            }
    return o;
}

static M part(const M& qkv, int from, int n) {  // heads [from, from + n) of a packed projection
    M out;
    for (int t = 0; t < B * T; ++t)
        out.insert(out.end(), qkv.begin() + (size_t(t) * (HQ + 2 * HK) + from) * D, qkv.begin() + (size_t(t) * (HQ + 2 * HK) + from + n) * D);
    return out;
}

int main() {
    const qsml::u32 b = B, t = T, hq = HQ, hk = HK, d = D;
    const M qkv = values(size_t(B) * T * (HQ + 2 * HK) * D, 1, 1.0), wq = values(D, 2, 0.2, 1), wk = values(D, 3, 0.2, 1);
    const M freq = {1.0f, 0.3f, 0.05f}, dout = values(size_t(B) * T * HQ * D, 4, 1.0);
    vector<int> pos(B * T);
    for (int i = 0; i < B * T; ++i) pos[i] = 100 * (i / T) + i % T;
    const M q = part(qkv, 0, HQ), k = part(qkv, HQ, HK), v = part(qkv, HQ + HK, HK);
    const M rq = norm_rotary(q, HQ, wq, freq, pos), rk = norm_rotary(k, HK, wk, freq, pos);
    const vector<int> all(B, T);
    Grads g{M(rq.size(), 0.0), M(rk.size(), 0.0), M(v.size(), 0.0)};
    const M o = attend(rq, rk, v, T, all, &dout, &g);
    M dwq(D, 0.0), dwk(D, 0.0);
    const M dq = norm_rotary(q, HQ, wq, freq, pos, &g.q, &dwq), dk = norm_rotary(k, HK, wk, freq, pos, &g.k, &dwk);

    auto packed = up(qkv, {b, t, hq + 2 * hk, d});
    auto tq = qsml::slice(packed, 2, 0, HQ), tk = qsml::slice(packed, 2, HQ, HQ + HK), tv = qsml::slice(packed, 2, HQ + HK, HQ + 2 * HK);
    auto twq = up(wq, {d}), twk = up(wk, {d}), tf = up(freq, {3}), tp = ints(pos, {b, t});
    auto r = qsml::norm_rotary(tq, tk, twq, twk, tp, tf);
    check("queries", close(r.q, rq));
    check("keys", close(r.k, rk));
    qsml::AttentionOptions opt;
    opt.window = W;
    opt.sinks = SINKS;
    TensorPtr lse;
    auto to = qsml::attention(r.q, r.k, tv, opt, &lse);
    check("attention", close(to, o));
    auto ga = qsml::attention_backward(r.q, r.k, tv, to, lse, up(dout, {b, t, hq, d}), opt);
    check("gradients of attention", close(ga.dq, g.q) && close(ga.dk, g.k) && close(ga.dv, g.v));
    auto gn = qsml::norm_rotary_backward(tq, tk, twq, twk, tp, tf, ga.dq, ga.dk);
    check("gradients of norm and rotation", close(gn.dq, dq) && close(gn.dk, dk) && close(gn.dwq, dwq) && close(gn.dwk, dwk));
    // the next token of two sequences of different lengths over a cache
    const vector<int> nk = {T, 7};
    M next;
    for (int s = 0; s < B; ++s)
        next.insert(next.end(), rq.begin() + (size_t(s) * T + nk[s] - 1) * HQ * D, rq.begin() + (size_t(s) * T + nk[s]) * HQ * D);
    opt.k_lengths = ints(nk, {b});
    check("next tokens", close(qsml::attention(up(next, {b, 1, hq, d}), r.k, tv, opt), attend(next, rk, v, 1, nk)));
    // transposed last dims are copied
    auto flipped = qsml::transpose(qsml::contiguous(qsml::transpose(r.q, 2, 3)), 2, 3);
    opt.k_lengths = nullptr;
    check("other layouts", close(qsml::attention(flipped, r.k, tv, opt), o));
    // queries alone, without a norm, by two axes
    qsml::RotaryOptions two;
    two.sections = {1, 2};
    vector<int> pos2;
    for (int p : pos) pos2.push_back(p), pos2.push_back(p);
    auto alone = qsml::norm_rotary(tq, nullptr, twq, nullptr, ints(pos2, {b, t, 2}), tf, two);
    check("axes", close(alone.q, rq) && !alone.k);
    auto throws = [](auto fn) {
        try {
            fn();
        } catch (const std::runtime_error&) {
            return true;
        }
        return false;
    };
    check("heads", throws([&] { qsml::attention(r.q, qsml::slice(packed, 2, 0, 3), qsml::slice(packed, 2, 0, 3)); }));
    check("sections", throws([&] { qsml::norm_rotary(tq, tk, twq, twk, tp, tf, two); }));
    check("null", throws([&] { qsml::attention(r.q, nullptr, tv); }));
    check("usable after errors", close(qsml::attention(r.q, r.k, tv, opt), o));
    qsml::shutdown();
    std::cout << "passed " << passed << " failed " << failed << "\n";
    return failed ? 1 : 0;
}
