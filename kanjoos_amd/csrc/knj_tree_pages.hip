// kanjoos_amd/csrc/knj_tree_pages.hip -- the drafts' attention (knj_tree.h) over 4-bit pages.
#include "knj_tree.h"

namespace knj {
namespace tree {

KNJ_TREE_FORMAT(kFormatPages)

}  // namespace tree
}  // namespace knj
