// What the entry points of the paged cache check alike: the cache's shape, and outputs that share memory.
#pragma once

#include <string.h>

#include <initializer_list>

#include "common.hpp"
#include "page_math.hpp"
#include "page_spans.hpp"

namespace pa {

// (paged.hip)
int check_pages(const char* who, int64_t n_pages, int32_t page_size, int* page_lg);

struct Named {
  const char* name;
  Strided<1> at;
  const char* same = "";  // an input that this output may be
};
inline Strided<1> tables_span(const int32_t* tables, int32_t R, int64_t pitch, int32_t cols) {
  return strided<1>(tables, 4ll * cols, {cols ? R : 0}, {pitch}, 4);
}
inline int check_apart(const char* who, std::initializer_list<Named> in, std::initializer_list<Named> out) {
  for (const Named& o : out) {
    for (const Named& i : in)
      PA_CHECK_ARG(!overlap(o.at, i.at) || (!strcmp(o.same, i.name) && o.at.at == i.at.at && span(o.at) == span(i.at)),
                   "%s: %s and %s overlap", who, o.name, i.name);
    for (const Named& i : out)
      PA_CHECK_ARG(&i == &o || !overlap(o.at, i.at), "%s: %s and %s overlap", who, o.name, i.name);
  }
  return PA_OK;
}

}  // namespace pa
