#include "book.h"

#include <algorithm>
#include <stdexcept>
#include <string>
#include <unordered_map>

namespace ddb {
namespace {
constexpr int64_t kPage = 64;
constexpr int64_t kMaxTokens = int64_t{1} << 30;
int64_t pages_of(int64_t tokens) { return (tokens + kPage - 1) / kPage; }
[[noreturn]] void refuse(const std::string& why) { throw std::invalid_argument(why); }
}  // namespace

KvBook::KvBook(int64_t pages, int64_t max_pages) : refs_(pages, 0), max_pages_(max_pages), free_(pages) {}

const KvBook::Seq& KvBook::seq(int64_t id) const {
  const auto it = seqs_.find(id);
  if (it == seqs_.end()) refuse("no sequence " + std::to_string(id) + " in this cache");
  return it->second;
}

std::vector<KvBook::Seq*> KvBook::get(const Ids& ids) {
  Ids sorted = ids;
  std::sort(sorted.begin(), sorted.end());
  if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end()) refuse("a sequence is named twice");
  std::vector<Seq*> out;
  out.reserve(ids.size());
  for (const int64_t id : ids) out.push_back(const_cast<Seq*>(&seq(id)));
  return out;
}

void KvBook::need(int64_t n) const {
  if (n > free_)
    throw std::runtime_error("out of cache pages: " + std::to_string(n) + " needed, " + std::to_string(free_) + " of " +
                             std::to_string(refs_.size()) + " free");
}

KvBook::Pages KvBook::take(int64_t n) {
  Pages out;
  out.reserve(n);
  for (; static_cast<int64_t>(out.size()) < n; ++low_)
    if (refs_[low_] == 0) {
      refs_[low_] = 1;
      out.push_back(static_cast<int32_t>(low_));
    }
  free_ -= n;
  return out;
}

void KvBook::give(int32_t page) {
  if (page < 0 || --refs_[page] > 0) return;
  ++free_;
  low_ = std::min<int64_t>(low_, page);
}

KvBook::Ids KvBook::add(int64_t n) {
  if (n < 0) refuse("n must not be negative");
  Ids out;
  for (int64_t i = 0; i < n; ++i) {
    seqs_.emplace_hint(seqs_.end(), next_, Seq{});
    out.push_back(next_++);
  }
  return out;
}

int64_t KvBook::longest(const Ids& ids, const Ids& n_new) const {
  int64_t most = 0;
  for (size_t i = 0; i < ids.size(); ++i) most = std::max(most, seq(ids[i]).length + n_new[i]);
  return most;
}

KvBook::Copies KvBook::begin(const Ids& ids, const Ids& n_new, int64_t max_tokens) {
  const auto states = get(ids);
  if (n_new.size() != ids.size() || std::any_of(n_new.begin(), n_new.end(), [](int64_t n) { return n < 0; }))
    refuse("n_new must be one number, or one for each sequence, none negative");
  if (std::any_of(n_new.begin(), n_new.end(), [](int64_t n) { return n > kMaxTokens; }))
    refuse("at most " + std::to_string(kMaxTokens) + " tokens");
  const int64_t most = longest(ids, n_new);
  if (most > max_pages_ * kPage)
    refuse(std::to_string(most) + " tokens do not fit a sequence's " + std::to_string(max_pages_) + " pages");
  if (max_tokens >= 0 && most > max_tokens)
    refuse("sequences of " + std::to_string(most) + " tokens in a step for " + std::to_string(max_tokens));
  // Pages to take: behind the present ones, and for shared pages that get new tokens (of a page
  // shared within this call the last one to write keeps it). Pages behind the new tokens are
  // the room of an abandoned step; they are given back first.
  int64_t more = 0;
  std::unordered_map<int32_t, int32_t> left;
  for (size_t i = 0; i < states.size(); ++i) {
    const Seq& s = *states[i];
    const int64_t have = s.pages.size(), upto = pages_of(s.length + n_new[i]);
    more += upto - have;
    for (int64_t j = s.length / kPage; n_new[i] > 0 && j < std::min(upto, have); ++j) {
      const int32_t p = s.pages[j];
      if (refs_[p] > 1 && --left.try_emplace(p, refs_[p]).first->second > 0) ++more;
    }
  }
  need(more);
  ++epoch;
  for (size_t i = 0; i < states.size(); ++i) {
    Seq& s = *states[i];
    const size_t upto = pages_of(s.length + n_new[i]);
    for (size_t j = upto; j < s.pages.size(); ++j) {
      give(s.pages[j]);
      ++more;
    }
    if (s.pages.size() > upto) s.pages.resize(upto);
  }
  const Pages fresh = take(more);
  size_t at = 0;
  Copies copies;
  for (size_t i = 0; i < states.size(); ++i) {
    Seq& s = *states[i];
    ++s.version;
    for (size_t j = s.length / kPage; n_new[i] > 0 && j < s.pages.size(); ++j) {
      const int32_t p = s.pages[j];
      if (refs_[p] <= 1) continue;
      --refs_[p];
      s.pages[j] = fresh[at++];
      if (static_cast<int64_t>(j) * kPage < s.length) {
        copies.src.push_back(p);
        copies.dst.push_back(s.pages[j]);
      }
    }
    const size_t upto = pages_of(s.length + n_new[i]), grown = upto - s.pages.size();
    s.pages.insert(s.pages.end(), fresh.begin() + at, fresh.begin() + at + grown);
    at += grown;
  }
  return copies;
}

void KvBook::commit(const Ids& ids, const Ids& n_new) {
  const auto states = get(ids);
  ++epoch;
  for (size_t i = 0; i < states.size(); ++i) {
    states[i]->length += n_new[i];
    ++states[i]->version;
  }
}

KvBook::Ids KvBook::fork(const Ids& ids, int64_t copies) {
  const auto states = get(ids);
  if (copies < 0) refuse("copies must not be negative");
  ++epoch;
  const Ids out = add(copies * static_cast<int64_t>(ids.size()));
  size_t at = 0;
  for (Seq* s : states) {
    ++s->version;
    Seq kid = *s;
    kid.pages.resize(pages_of(s->length));
    kid.version = 0;
    for (const int32_t p : kid.pages)
      if (p >= 0) refs_[p] += static_cast<int32_t>(copies);
    for (int64_t c = 0; c < copies; ++c) seqs_.at(out[at++]) = kid;
  }
  return out;
}

std::pair<KvBook::Ids, KvBook::Copies> KvBook::copy(const Ids& ids) {
  const auto states = get(ids);
  Copies copies;
  for (const Seq* s : states)
    for (int64_t j = 0; j < pages_of(s->length); ++j)
      if (s->pages[j] >= 0) copies.src.push_back(s->pages[j]);
  need(copies.src.size());
  copies.dst = take(copies.src.size());
  const Ids out = add(ids.size());
  size_t at = 0;
  for (size_t i = 0; i < states.size(); ++i) {
    Seq twin = *states[i];
    twin.pages.resize(pages_of(twin.length));
    twin.version = 0;
    for (int32_t& p : twin.pages)
      if (p >= 0) p = copies.dst[at++];
    seqs_.at(out[i]) = std::move(twin);
  }
  return {out, std::move(copies)};
}

void KvBook::free(const Ids& ids) {
  const auto states = get(ids);
  if (ids.empty()) return;
  ++epoch;
  for (const Seq* s : states)
    for (const int32_t p : s->pages) give(p);
  for (const int64_t id : ids) seqs_.erase(id);
}

void KvBook::trim(const Ids& ids, int64_t keep, int64_t sinks) {
  const auto states = get(ids);
  if (keep < 0 || sinks < 0) refuse("keep and sinks must not be negative");
  keep = std::min(keep, kMaxTokens);
  sinks = std::min(sinks, kMaxTokens);
  for (const Seq* s : states)
    if (s->trimmed() && s->sinks != sinks) refuse("a sequence that was trimmed keeps its number of sinks");
  ++epoch;
  for (Seq* s : states) {
    const int64_t first = std::max(s->first, s->length - keep);
    if (first <= sinks) continue;
    // pages up to the old `first` went before
    const int64_t lo = std::max(pages_of(sinks), s->trimmed() ? s->first / kPage : 0);
    for (int64_t j = lo; j < first / kPage; ++j) {
      give(s->pages[j]);
      s->pages[j] = -1;
    }
    s->first = first;
    s->sinks = sinks;
    ++s->version;
  }
}

KvBook::Copies KvBook::compact() {
  const int64_t n = static_cast<int64_t>(refs_.size()) - free_;
  Copies moves;
  for (int64_t p = 0; p < static_cast<int64_t>(refs_.size()); ++p) {
    if (p < n && refs_[p] == 0) moves.dst.push_back(static_cast<int32_t>(p));
    if (p >= n && refs_[p] > 0) moves.src.push_back(static_cast<int32_t>(p));
  }
  if (moves.src.empty()) return moves;
  ++epoch;
  std::unordered_map<int32_t, int32_t> to;
  for (size_t i = 0; i < moves.src.size(); ++i) {
    to[moves.src[i]] = moves.dst[i];
    std::swap(refs_[moves.dst[i]], refs_[moves.src[i]]);
  }
  for (auto& [id, s] : seqs_) {
    bool moved = false;
    for (int32_t& p : s.pages)
      if (p >= n) {
        p = to.at(p);
        moved = true;
      }
    s.version += moved;
  }
  low_ = n;
  return moves;
}

int64_t KvBook::used_end() const {
  int64_t p = refs_.size();
  while (p > 0 && refs_[p - 1] == 0) --p;
  return p;
}

void KvBook::resize(int64_t pages, int64_t max_pages) {
  if (pages < used_end()) refuse("pages behind the new size are in use");
  max_pages_ = std::max(max_pages_, max_pages);
  free_ += pages - static_cast<int64_t>(refs_.size());
  refs_.resize(pages, 0);
  low_ = 0;
  ++epoch;
  for (auto& [id, s] : seqs_) ++s.version;
}

int64_t KvBook::trim_sinks(const Ids& ids) const {
  int64_t trim = -1;
  for (const int64_t id : ids) {
    const Seq& s = seq(id);
    if (s.trimmed()) trim = trim == -1 || trim == s.sinks ? s.sinks : -2;
  }
  return trim;
}

void KvBook::rows(const Ids& ids, const Ids& n_new, int front, int32_t* out) const {
  for (size_t i = 0; i < ids.size(); ++i) {
    const Seq& s = seq(ids[i]);
    if (front == kFront) {
      out[0] = static_cast<int32_t>(s.length + n_new[i]);
      out[1] = static_cast<int32_t>(n_new[i]);
      out[2] = s.trimmed() ? static_cast<int32_t>(s.first) : 0;
      out[3] = s.trimmed() ? static_cast<int32_t>(s.sinks) : -1;
    }
    out = std::copy(s.pages.begin(), s.pages.end(), out + front);
    out = std::fill_n(out, max_pages_ - static_cast<int64_t>(s.pages.size()), -1);
  }
}

std::pair<int64_t, int64_t> KvBook::shared_rows(const Ids& ids, const Ids& n_new, int64_t branches, int32_t* out) const {
  int64_t most = 0, own = 0;
  for (size_t i = 0; i < ids.size(); i += branches) {
    std::vector<const Seq*> group;
    int64_t n = max_pages_;
    for (int64_t k = 0; k < branches; ++k) {
      group.push_back(&seq(ids[i + k]));
      n = std::min(n, group[k]->length / kPage);
    }
    int32_t* pages = out + kFront;
    std::copy_n(group[0]->pages.begin(), n, pages);
    for (const Seq* s : group) {
      if (std::equal(pages, pages + n, s->pages.begin())) continue;
      for (int64_t j = 0; j < n; ++j) {  // a page that one sequence gave back is hidden from it alone
        const int32_t p = s->pages[j];
        if (pages[j] < 0) pages[j] = p;
        else if (p >= 0 && p != pages[j]) n = j;
      }
    }
    std::fill_n(out, kFront, 0);
    out[0] = static_cast<int32_t>(n);
    std::fill_n(pages + n, max_pages_ - n, -1);
    out += kFront + max_pages_;
    most = std::max(most, n);
    for (int64_t k = 0; k < branches; ++k) own = std::max(own, group[k]->length + n_new[i + k] - n * kPage);
  }
  return {most, own};
}

KvBook::Ids KvBook::versions(const Ids& ids) const {
  Ids out;
  out.reserve(ids.size());
  for (const int64_t id : ids) out.push_back(seq(id).version);
  return out;
}

bool KvBook::fresh(const Ids& ids, const Ids& versions) const {
  for (size_t i = 0; i < ids.size(); ++i) {
    const auto it = seqs_.find(ids[i]);
    if (it == seqs_.end() || it->second.version != versions[i]) return false;
  }
  return true;
}

}  // namespace ddb
