// Host bookkeeping of the paged cache: the sequences, the pages that each holds in order, and
// how many sequences hold each page. No device work; calls come from one thread. A call
// that cannot be met throws (std::invalid_argument for its arguments, std::runtime_error
// when pages run out) before it changes anything.
#pragma once
#include <cstdint>
#include <map>
#include <utility>
#include <vector>

namespace ddb {

class KvBook {
 public:
  using Ids = std::vector<int64_t>;
  using Pages = std::vector<int32_t>;
  static constexpr int kFront = 4;  // words of a step's row before its page ids (kvcache.h)

  struct Seq {
    Pages pages;          // by page of the sequence; -1: given back
    int64_t length = 0;   // committed tokens
    int64_t first = 0;    // tokens in [sinks, first) are gone
    int64_t sinks = 0;
    int64_t version = 0;  // a step begun at another version is stale
    bool trimmed() const { return first > sinks; }
  };
  struct Copies {         // pages to copy, of every layer
    Pages src, dst;
  };

  KvBook(int64_t pages, int64_t max_pages);

  Ids add(int64_t n);
  // Room for n_new[i] tokens behind each sequence; max_tokens -1: any length. A shared
  // unfinished page that gets tokens is replaced by a copy.
  Copies begin(const Ids& seqs, const Ids& n_new, int64_t max_tokens);
  void commit(const Ids& seqs, const Ids& n_new);
  Ids fork(const Ids& seqs, int64_t copies);
  std::pair<Ids, Copies> copy(const Ids& seqs);
  void free(const Ids& seqs);
  void trim(const Ids& seqs, int64_t keep, int64_t sinks);
  Copies compact();
  void resize(int64_t pages, int64_t max_pages);  // max_pages does not shrink

  // A step's table, [sequences][front + max_pages]: front kFront writes the words that precede
  // the page ids too, 0 the ids alone.
  void rows(const Ids& seqs, const Ids& n_new, int front, int32_t* out) const;
  // The pages that groups of `branches` consecutive sequences share, [groups][kFront + max_pages]: how
  // many leading pages lie behind no sequence's new tokens and are the same for all that still have
  // them, then their ids (-1: none has it). Returns the most such pages of a group, and the most
  // tokens of a sequence behind its group's.
  std::pair<int64_t, int64_t> shared_rows(const Ids& seqs, const Ids& n_new, int64_t branches, int32_t* out) const;
  // the sinks of the trimmed sequences (-1: none is, -2: they differ)
  int64_t trim_sinks(const Ids& seqs) const;
  int64_t longest(const Ids& seqs, const Ids& n_new) const;
  Ids versions(const Ids& seqs) const;
  bool fresh(const Ids& seqs, const Ids& versions) const;
  const Seq& seq(int64_t id) const;

  const std::map<int64_t, Seq>& seqs() const { return seqs_; }
  const Pages& refs() const { return refs_; }
  int64_t free_pages() const { return free_; }
  int64_t max_pages() const { return max_pages_; }
  int64_t used_end() const;  // behind the last page in use
  int64_t epoch = 0;         // counts changes of any sequence

 private:
  std::vector<Seq*> get(const Ids& seqs);
  void need(int64_t n) const;
  Pages take(int64_t n);     // the n lowest free pages (there are as many)
  void give(int32_t page);   // one sequence's hold of a page ends

  Pages refs_;               // sequences that hold a page
  int64_t max_pages_, free_, low_ = 0;  // no page below low_ is free
  std::map<int64_t, Seq> seqs_;
  int64_t next_ = 0;
};

}  // namespace ddb
