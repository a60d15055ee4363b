# The host code of chunk attention and shared pages under AddressSanitizer and
# UndefinedBehaviorSanitizer, linked into kvq_share_check (as pages.mk does).
include $(dir $(abspath $(lastword $(MAKEFILE_LIST))))Makefile
.DEFAULT_GOAL := share
SHARE := $(foreach n,kvq_share kvq_chunk kvq_share_capi,$(BUILD)/$(n).o)

share: $(BUILD)/kvq_share_check

$(BUILD)/kvq_share_capi.o: $(CSRC)/kvq_share_capi.cpp $(DEPS)
	@mkdir -p $(BUILD)
	$(HIPCC) $(FLAGS) -c $< -o $@

$(BUILD)/kvq_share_check.o: $(HERE)kvq_share_check.cpp $(DEPS)
	@mkdir -p $(BUILD)
	$(HIPCC) $(FLAGS) -c $< -o $@

$(BUILD)/kvq_share_check: $(OBJS) $(SHARE) $(BUILD)/kvq_share_check.o
	$(HIPCC) --offload-arch=gfx950 $(SAN) -o $@.tmp $^ && mv $@.tmp $@

.PHONY: share
