// storage_base.h — test-side stand-in for the reference's tinytensor/tensor/storage_base.h (see backend_base.h beside it).
#ifndef TT_STANDIN_STORAGE_BASE_H_
#define TT_STANDIN_STORAGE_BASE_H_

namespace tinytensor {

class StorageBase {
public:
    virtual ~StorageBase() = default;
};

}  // namespace tinytensor

#endif  // TT_STANDIN_STORAGE_BASE_H_
