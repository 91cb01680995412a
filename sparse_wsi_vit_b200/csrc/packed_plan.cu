// Host side of the packed attention: turns the lengths of the sequences of a batch into the kernels' work tables.
//
// A unit is what one CTA does: two tiles of 128 (query, head of the group) rows against the keys that they see in the
// forward pass, one such tile in the dq pass, 128 keys against the queries that see them in the dkv pass.  Units are
// sorted by their work, the longest first, so that the last CTAs of a launch are the short ones.
//
// Where the units are few, long ones are divided: how often is found by laying candidates out over the SMs the way
// the hardware does (the next unit to the SM that is free first) and taking the one that ends first.  (Only units of three blocks
// and more are divided: the forward join relies on it.)  A unit costs its
// blocks and two more for its start and end, a divided one a further block to leave its sums and read them back; the
// join launch costs three.
#include <algorithm>
#include <cstring>
#include <queue>
#include <vector>

#include "packed.cuh"

namespace swv {
namespace {

struct Work {
  std::vector<PackedUnit> units;
  std::vector<PackedJoin> joins;
  int slots = 0;
};

int64_t makespan(const std::vector<PackedUnit>& units, int heads, int chunk, int sms, int64_t behind) {
  std::vector<int> cost;
  bool divided = false;
  for (const PackedUnit& u : units) {
    const int n = u.b1 - u.b0, parts = n > chunk ? (n + chunk - 1) / chunk : 1;
    divided |= parts > 1;
    for (int i = 0; i < parts; ++i)
      for (int h = 0; h < heads; ++h) cost.push_back((n + parts - 1) / parts + 2 + (parts > 1 ? 1 : 0));
  }
  std::sort(cost.begin(), cost.end(), [](int a, int b) { return a > b; });
  std::priority_queue<int64_t, std::vector<int64_t>, std::greater<int64_t>> free_at;
  for (int i = 0; i < sms; ++i) free_at.push(0);
  int64_t end = 0, sum = behind;
  for (int c : cost) {
    sum += c;
    const int64_t t = free_at.top() + c;
    free_at.pop();
    free_at.push(t);
    end = std::max(end, t);
  }
  return std::max(end, sum / sms) + (divided ? 3 : 0);
}

int64_t total(const Work& w, int heads) {
  int64_t sum = 0;
  for (const PackedUnit& u : w.units) sum += u.b1 - u.b0 + 2;
  return sum * heads;
}

// divides the units (all of `heads` heads each) and sorts them; `behind`: the work of the CTAs behind them in the grid, which fill the SMs
// that they leave free, so that they need not end together (keys' side of 8192 causal tokens, 16 heads of 128 sharing two key heads:
// 128 instead of 430 partial sums, training pass 1035 -> 1005 us)
void divide(Work& w, int heads, int sms, int64_t behind = 0) {
  int longest = 0;
  for (const PackedUnit& u : w.units) longest = std::max(longest, u.b1 - u.b0);
  int best_chunk = std::max(longest, 1);
  // (with four units an SM no unit is long against the whole)
  if (longest > 2 && static_cast<int64_t>(w.units.size()) * heads < 4ll * sms) {
    int64_t best = makespan(w.units, heads, best_chunk, sms, behind);
    for (int parts = 2; parts <= 128; parts += std::max(1, parts / 4)) {
      const int chunk = std::max(2, (longest + parts - 1) / parts);
      const int64_t t = makespan(w.units, heads, chunk, sms, behind);
      if (t < best) {
        best = t;
        best_chunk = chunk;
      }
      int64_t pieces = 0;
      for (const PackedUnit& u : w.units) pieces += std::max(1, (u.b1 - u.b0 + chunk - 1) / chunk);
      if (chunk == 2 || pieces * heads > 8ll * sms) break;          // finer pieces only add their own cost
    }
  }
  std::vector<PackedUnit> out;
  for (const PackedUnit& u : w.units) {
    const int n = u.b1 - u.b0, parts = n > best_chunk ? (n + best_chunk - 1) / best_chunk : 1;
    if (parts > 1) w.joins.push_back({u.t0, u.n, w.slots, parts});
    for (int i = 0; i < parts; ++i) {
      PackedUnit v = u;
      v.b0 = u.b0 + static_cast<int>(static_cast<int64_t>(n) * i / parts);
      v.b1 = u.b0 + static_cast<int>(static_cast<int64_t>(n) * (i + 1) / parts);
      v.slot = parts > 1 ? w.slots++ : -1;
      out.push_back(v);
    }
  }
  std::stable_sort(out.begin(), out.end(),
                   [](const PackedUnit& a, const PackedUnit& b) { return a.b1 - a.b0 > b.b1 - b.b0; });
  w.units.swap(out);
}

int check(int n_seq, const int64_t* ql, const int64_t* kl, int H, int Hkv, int64_t* Tq, int64_t* Tk) {
  if (n_seq < 0 || H < 1 || Hkv < 1 || H % Hkv != 0) return SWV_ERR_SHAPE;
  if (n_seq > 0 && (!ql || !kl)) return SWV_ERR_NULL;
  if (H / Hkv > kTile) return SWV_ERR_UNSUPPORTED;
  *Tq = *Tk = 0;
  const int64_t tok = kTile / (H / Hkv);
  int64_t units = 0;                              // of the three passes
  for (int i = 0; i < n_seq; ++i) {
    if (ql[i] < 0 || kl[i] < 0) return SWV_ERR_SHAPE;
    *Tq += ql[i];
    *Tk += kl[i];
    // token indices, key limits and their sums stay within 32 bits
    if (*Tq > (1 << 29) || *Tk > (1 << 29)) return SWV_ERR_UNSUPPORTED;
    // and so do the tables' offsets in words (eight a unit; dividing adds few)
    units += (ql[i] + 2 * tok - 1) / (2 * tok) + (ql[i] + tok - 1) / tok + (kl[i] + kTile - 1) / kTile;
    if (units > (1 << 27)) return SWV_ERR_UNSUPPORTED;
  }
  return SWV_OK;
}

void build(int n_seq, const int64_t* ql, const int64_t* kl, int H, int Hkv, int causal, std::vector<int>& out) {
  const int tok = kTile / (H / Hkv);              // query tokens of a tile
  const int sms = sm_count();
  Work fwd, dq, dkv;
  int q0 = 0, k0 = 0, longest_q = 0, longest_k = 0;
  for (int s = 0; s < n_seq; ++s) {
    const int lq = static_cast<int>(ql[s]), lk = static_cast<int>(kl[s]);
    for (int pass = 0; pass < 2; ++pass) {
      Work& w = pass == 0 ? fwd : dq;
      const int step = pass == 0 ? 2 * tok : tok;
      for (int t = 0; t < lq; t += step) {
        PackedUnit u;
        u.t0 = q0 + t;
        u.n = std::min(step, lq - t);
        u.s0 = k0;
        u.len = lk;
        u.off = causal ? t + lk - lq : lk;
        const int sees = std::max(0, std::min(lk, u.off + u.n));     // keys that the unit's last token sees
        u.b0 = 0;
        u.b1 = (sees + kTile - 1) / kTile;
        u.slot = -1;
        w.units.push_back(u);
      }
    }
    for (int t = 0; t < lk; t += kTile) {
      PackedUnit u;
      u.t0 = k0 + t;
      u.n = std::min(kTile, lk - t);
      u.s0 = q0;
      u.len = lq;
      u.off = causal ? t - (lk - lq) : -kTile;                       // key i is seen by queries j >= off + i
      const int first = std::max(0, u.off);
      u.b1 = (lq + tok - 1) / tok;
      u.b0 = std::min(first / tok, u.b1);
      u.slot = -1;
      dkv.units.push_back(u);
    }
    longest_q = std::max(longest_q, lq);
    longest_k = std::max(longest_k, lk);
    q0 += lq;
    k0 += lk;
  }
  divide(fwd, Hkv, sms);
  divide(dq, Hkv, sms);
  divide(dkv, Hkv, sms, total(dq, Hkv));                      // (the queries' side follows in the same grid)
  PackedHeader h{};
  h.magic = kPlanMagic;
  h.n_seq = n_seq; h.H = H; h.Hkv = Hkv; h.causal = causal; h.Tq = q0; h.Tk = k0;
  h.longest_q = longest_q; h.longest_k = longest_k;
  out.assign(kPlanHeader, 0);
  auto put = [&](const Work& w, int& off, int& n, int& join_off, int& n_join, int& slots) {
    off = static_cast<int>(out.size());
    n = static_cast<int>(w.units.size());
    out.resize(out.size() + w.units.size() * 8);
    if (n) memcpy(out.data() + off, w.units.data(), w.units.size() * sizeof(PackedUnit));
    join_off = static_cast<int>(out.size());
    n_join = static_cast<int>(w.joins.size());
    out.resize(out.size() + w.joins.size() * 4);
    if (n_join) memcpy(out.data() + join_off, w.joins.data(), w.joins.size() * sizeof(PackedJoin));
    while (out.size() % 8) out.push_back(0);      // units start on 32 bytes
    slots = w.slots;
  };
  put(fwd, h.fwd_off, h.n_fwd, h.fwd_join_off, h.n_fwd_join, h.fwd_slots);
  put(dq, h.dq_off, h.n_dq, h.dq_join_off, h.n_dq_join, h.dq_slots);
  put(dkv, h.dkv_off, h.n_dkv, h.dkv_join_off, h.n_dkv_join, h.dkv_slots);
  h.words = static_cast<int>(out.size());
  memcpy(out.data(), &h, sizeof(h));
}

}  // namespace

int packed_plan_impl(int n_seq, const int64_t* q_lens, const int64_t* k_lens, int H, int Hkv, int causal, int32_t* plan,
                     size_t plan_bytes, size_t* bytes) {
  if (plan == nullptr && bytes == nullptr) return SWV_ERR_NULL;
  int64_t Tq = 0, Tk = 0;
  const int rc = check(n_seq, q_lens, k_lens, H, Hkv, &Tq, &Tk);
  if (rc != SWV_OK) return rc;
  try {
    std::vector<int> out;
    build(n_seq, q_lens, k_lens, H, Hkv, causal != 0, out);
    if (bytes != nullptr) *bytes = out.size() * 4;
    if (plan != nullptr) {
      if (plan_bytes < out.size() * 4) return SWV_ERR_WORKSPACE;
      memcpy(plan, out.data(), out.size() * 4);
    }
  } catch (...) {                                 // (host memory ran out)
    return SWV_ERR_UNSUPPORTED;
  }
  return SWV_OK;
}

}  // namespace swv
