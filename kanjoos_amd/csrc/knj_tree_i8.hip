// kanjoos_amd/csrc/knj_tree_i8.hip -- the drafts' attention (knj_tree.h) over a KNJ_KV_I8 cache.
#include "knj_tree.h"

namespace knj {
namespace tree {

KNJ_TREE_FORMAT(KNJ_KV_I8)

}  // namespace tree
}  // namespace knj
