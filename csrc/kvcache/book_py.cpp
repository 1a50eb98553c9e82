// Python bindings of the paged cache's bookkeeping. They are in the host-only extension: a cache on
// the CPU needs no CUDA one.
#include <pybind11/numpy.h>
#include <torch/extension.h>

#include "book.h"

namespace py = pybind11;

namespace {

torch::Tensor host_ints(const std::vector<int32_t>& v) {
  auto t = torch::empty({static_cast<int64_t>(v.size())}, torch::kInt32);
  std::copy(v.begin(), v.end(), t.data_ptr<int>());
  return t;
}

// (step rows, behind them those of the groups' shared pages; pages to copy from, to, longest sequence,
// sinks of the trimmed ones, versions, most shared pages, most tokens behind them)
py::tuple kv_book_begin(ddb::KvBook& book, const ddb::KvBook::Ids& seqs, const ddb::KvBook::Ids& n_new, int64_t max_tokens,
                        int64_t branches) {
  const int64_t n = seqs.size();
  if (branches < 1 || n % branches) throw std::invalid_argument("the sequences are no whole groups of branches");
  const auto copies = book.begin(seqs, n_new, max_tokens);
  const int64_t groups = branches > 1 ? n / branches : 0, ld = ddb::KvBook::kFront + book.max_pages();
  auto rows = torch::empty({n + groups, ld}, torch::kInt32);
  book.rows(seqs, n_new, ddb::KvBook::kFront, rows.data_ptr<int>());
  const auto shared = groups ? book.shared_rows(seqs, n_new, branches, rows.data_ptr<int>() + n * ld) : std::pair<int64_t, int64_t>{0, 0};
  return py::make_tuple(rows, host_ints(copies.src), host_ints(copies.dst), book.longest(seqs, n_new), book.trim_sinks(seqs),
                        book.versions(seqs), shared.first, shared.second);
}
torch::Tensor kv_book_table(const ddb::KvBook& book, const ddb::KvBook::Ids& seqs) {
  auto rows = torch::empty({static_cast<int64_t>(seqs.size()), book.max_pages()}, torch::kInt32);
  book.rows(seqs, {}, 0, rows.data_ptr<int>());
  return rows;
}

}  // namespace

namespace ddb {

void bind_kv_book(py::module_& m) {
  py::class_<ddb::KvBook::Seq>(m, "KvSeq")
      .def_property_readonly("pages", [](const ddb::KvBook::Seq& s) { return py::array_t<int32_t>(s.pages.size(), s.pages.data()); })
      .def_readonly("length", &ddb::KvBook::Seq::length)
      .def_readonly("first", &ddb::KvBook::Seq::first)
      .def_readonly("sinks", &ddb::KvBook::Seq::sinks)
      .def_readonly("version", &ddb::KvBook::Seq::version)
      .def_property_readonly("trimmed", &ddb::KvBook::Seq::trimmed);
  py::class_<ddb::KvBook>(m, "KvBook")
      .def(py::init<int64_t, int64_t>())
      .def("add", &ddb::KvBook::add)
      .def("begin", &kv_book_begin)
      .def("commit", &ddb::KvBook::commit)
      .def("fork", &ddb::KvBook::fork)
      .def("copy", [](ddb::KvBook& b, const ddb::KvBook::Ids& seqs) {
        const auto made = b.copy(seqs);
        return py::make_tuple(made.first, host_ints(made.second.src), host_ints(made.second.dst));
      })
      .def("free", &ddb::KvBook::free)
      .def("trim", &ddb::KvBook::trim)
      .def("compact", [](ddb::KvBook& b) {
        const auto moves = b.compact();
        return py::make_tuple(host_ints(moves.src), host_ints(moves.dst));
      })
      .def("resize", &ddb::KvBook::resize)
      .def("table", &kv_book_table)
      .def("fresh", &ddb::KvBook::fresh)
      .def("trim_sinks", &ddb::KvBook::trim_sinks)
      .def("seq", &ddb::KvBook::seq, py::return_value_policy::copy)
      .def("seqs", &ddb::KvBook::seqs, py::return_value_policy::copy)
      .def("refs", [](const ddb::KvBook& b) { return py::array_t<int32_t>(b.refs().size(), b.refs().data()); })
      .def("used_end", &ddb::KvBook::used_end)
      .def_property_readonly("free_pages", &ddb::KvBook::free_pages)
      .def_readonly("epoch", &ddb::KvBook::epoch);
}

}  // namespace ddb
